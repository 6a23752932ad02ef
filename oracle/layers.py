"""Test infrastructure: the layer operators (mmvae_amd.ops) in 64 bits on the CPU, from their formulas.

The reference has no such layers; these are the definitions the operators' documentation states, with
the error bounds that 32-bit evaluation of them has."""
import numpy as np
import torch
import torch.nn.functional as F

from . import nb_oracle, philox, vmf_oracle

U32 = 2.0 ** -24  # half a step of float32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def drop_threshold(p):
    return int(np.floor(p * 65536 + 0.5))


def drop_kept(M, N, p, seed, step=0, row_offset=0):
    """The kept elements [M, N]: half col % 8 of philox(col / 8, row, step, step >> 32 ^ row >> 32) >= threshold."""
    rows = (np.arange(M, dtype=np.uint64) + np.uint64(row_offset))[:, None]
    grp = np.arange((N + 7) // 8, dtype=np.uint64)[None, :]
    shape = (M, grp.shape[1])
    seed, step = seed % 2 ** 64, step % 2 ** 64
    c = philox._philox4x32_10(np.broadcast_to(grp, shape), np.broadcast_to(rows & np.uint64(0xFFFFFFFF), shape),
                              np.full(shape, np.uint64(step & 0xFFFFFFFF)),
                              np.broadcast_to((rows >> np.uint64(32)) ^ np.uint64(step >> 32), shape),
                              seed & 0xFFFFFFFF, seed >> 32)
    halves = np.stack([h for w in c for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], axis=2)
    return torch.from_numpy(halves.reshape(M, -1)[:, :N] >= drop_threshold(p))


def drop_scale(p):
    t = drop_threshold(p)
    return 65536 / (65536 - t) if t < 65536 else 0.0


def drop_factor(M, N, p, seed, step=0, row_offset=0):
    return torch.where(drop_kept(M, N, p, seed, step, row_offset), drop_scale(p), 0.0).double() if p > 0 else torch.ones(M, N).double()


def norm(x, w, b, eps, factor, relu):
    """y, mean, rstd, u (before ReLU and dropout) of float64 tensors."""
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    u = (x - mean) * rstd * w + b
    y = (u.clamp(min=0) if relu else u) * factor
    return y, mean[:, 0], rstd[:, 0], u


def column_chain(M, N):
    """Additions in a column's sum over M rows, with room.  In strips: a thread's rows (M / 512, or up to 4), 6 lane steps, 8
    waves; in parts: a thread's rows (M / 256 at most), 32 row groups, a stage of 16 and one of 32; of rows that may be read
    in sweeps: 128 stripes of rows and two stages."""
    return M / (128 if N > 20480 else 256) + 96


def norm_grads(dy, x, w, eps, factor, mask):
    """dx, dw, db and the error bounds of their 32-bit evaluation (before the final rounding), with the ReLU's mask."""
    M, N = x.shape
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    du = dy * factor * mask
    g = du * w
    c1, c2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = rstd * (g - c1 - xh * c2)
    # A row's sums are chains of at most ROW additions, so the mean is off by ROW u mean|x|, xh by
    # ROW u A with A = rstd mean|x| + |xh| + 1, and the means of g and g xh by ROW u of their absolute sums.
    # (First order: for ROW u A well below 1, means up to some 10^4 times the spread.)
    a = rstd * x.abs().mean(1, keepdim=True) + xh.abs() + 1
    ag = (g.abs() * a).mean(1, keepdim=True)
    bdx = ROW * U32 * rstd * (2 * g.abs() + 2 * g.abs().mean(1, keepdim=True) + 2 * a * (g * xh).abs().mean(1, keepdim=True) + xh.abs() * 2 * ag)
    dw, db = (du * xh).sum(0), du.sum(0)
    col = column_chain(M, N)
    return dx, dw, db, bdx, U32 * ((col + ROW) * (du.abs() * a).sum(0)), U32 * col * du.abs().sum(0)


# Additions in a row's sum, with room: 8 elements of a chunk, a thread's up to 8 chunks, 6 lane steps, 8 waves; in sweeps
# (N > 32768) 8 + N / 8192 + 6 + 16.  The backward's two sums are chains of up to 8 x 8 + 14: the 2 in bdx covers them.
ROW = 72


def norm_bound(x, w, b, eps, factor):
    """The error bound of y before its final rounding: xh as above, times |w|, and the roundings of u."""
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    a = rstd * x.abs().mean(1, keepdim=True) + xh.abs() + 1
    return U32 * (ROW * a * w.abs() + 2 * b.abs()) * factor


def embedding(ids, table, scale, add=None):
    ok = (ids >= 0) & (ids < table.shape[0])
    y = torch.where(ok[..., None], table[torch.where(ok, ids, 0)] * scale, 0.0) if table.shape[0] else torch.zeros(*ids.shape, table.shape[1]).double()
    return y if add is None else y + add


def embedding_chain(T, N, rows):
    """Additions from a token's dy to its row of the gradient: its group's tokens, the piece's groups, a share of the pieces
    and the shares.  gb groups of tg tokens are a piece; 8, 16 or 32 lanes a row of N."""
    nc = (N + 7) // 8
    lanes = 8 if nc <= 8 else 16 if 5 * (-(-nc // 32) * 32) > 6 * (-(-nc // 16) * 16) else 32
    gb = 256 // lanes
    tg = 8 if T <= 32768 else 512 // gb if rows <= 64 else 16
    return tg + gb + -(-T // (gb * tg)) // gb + 1 + gb


def longest_chain(T, gb, tg, few):
    """dy of T tokens of one id whose 32-bit sum loses nearly half a step of 1 in every addition: 1, then addends just below
    2^-24 along one chain (sorted: a share of the pieces behind the first; few rows: a group, its piece, a share, the shares)."""
    d, P = torch.zeros(T), gb * tg
    tiny = 0.999 * U32
    if few:
        d[1:tg] = tiny
        d[tg:P:tg] = tiny
        d[P:gb * P:P] = tiny
        d[gb * P::gb * P] = tiny
        d[0] = 1
    else:
        d[P + gb * P::gb * P] = tiny
        d[P] = 1
    return d


def embedding_grad(dy, ids, rows, scale):
    """The table's gradient and the bound of its 32-bit sum: n additions and the scale's rounding, (1 + u)^(n + 1) - 1."""
    ok = (ids >= 0) & (ids < rows)
    i = torch.where(ok, ids, rows).reshape(-1).long()
    d = dy.reshape(-1, dy.shape[-1])
    out = torch.zeros(rows + 1, d.shape[1]).double().index_add_(0, i, d)
    mag = torch.zeros(rows + 1, d.shape[1]).double().index_add_(0, i, d.abs())
    n = embedding_chain(d.shape[0], d.shape[1], rows) + 1
    return out[:rows] * scale, n * U32 / (1 - n * U32) * abs(scale) * mag[:rows]


# ---- the models with normalised, dropped-out, label-conditioned layer chains --------------------
class _Chains:
    """The layer chains of a model oracle with cfg.layer_norm / dropout / n_labels.  `key` = (seed, step,
    row_offset) of the step; params hold the norms' weights and the label table under their names."""
    layer_norm, dropout, label_scale, labels, key, training = False, 0.0, 1.0, None, (42, 0, 0), True

    def _after(self, x, seq, l, relu):
        seed, step, ro = self.key
        if self.layer_norm:
            n = f"{self.prefix}{seq}.norm_{l + 1}"
            x = F.layer_norm(x, (x.shape[1],), self.p[n + ".weight"], self.p[n + ".bias"], 1e-5)
        if relu:
            x = F.relu(x)
        if self.dropout > 0 and self.training:
            k = seed + 0x9E3779B97F4A7C15 * ((1 if seq == "enc" else 101) + l)
            x = x * drop_factor(*x.shape, float(np.float32(self.dropout)), k, step, ro).to(x.dtype)
        return x

    def _z(self, z):
        if self.labels is None:
            return z
        t = self.p["label_embedding.weight"]
        ok = (self.labels >= 0)[:, None]
        return z + self.label_scale * torch.where(ok, t[self.labels.clamp(min=0)], torch.zeros_like(z))


class NBLayers(_Chains, nb_oracle.NBModel):
    prefix = "mu_"

    def _seq(self, keys, x, final_relu):
        enc = keys is self.enc_keys
        if not enc:
            x = self._z(x)
        for i, k in enumerate(keys):
            x = F.linear(x, self.fr[k + ".weight"], self.fr[k + ".bias"])
            last = i == len(keys) - 1
            if enc or not last:
                x = self._after(x, "enc" if enc else "dec", i, self.relu and (not last or final_relu))
        return x


class VMFLayers(_Chains, vmf_oracle.VMFModel):
    prefix = "z_"

    def z_enc(self, x):
        for i, k in enumerate(self.enc_keys):
            x = self._after(self.angular(x, k), "enc", i, self.relu)
        return x

    def z_dec(self, z):
        z = self._z(z)
        for i, k in enumerate(self.dec_keys):
            z = F.linear(z, self.fr[k + ".weight"], self.fr[k + ".bias"])
            if i < len(self.dec_keys) - 1:
                z = self._after(z, "dec", i, self.relu)
        return z
