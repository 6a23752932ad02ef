"""CPU tests of the layer operators' boundary (include/mmvae_capi.h, mmvae_amd.ops): the packed argument
structs match the header's, every wrong call is refused before a device is touched, the oracle's own
formulas hold against differences, and the dropout masks have the stated rate."""
import gzip
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import mmvae_amd
from mmvae_amd import host, ops
from oracle import layers

INCLUDE = os.path.dirname(mmvae_amd.HEADER_PATH)


def pack_norm(**kw):
    v = dict(M=4, N=8, x=4096, ldx=8, w=0, b=0, y=4096, ldy=8, mean=4096, rstd=4096, dy=4096, lddy=8, dx=4096, lddx=8, dw=4096, db=4096,
             ws=4096, ws_bytes=1 << 30, p=0.0, seed=1, step=0, row_offset=0, state=0, stream=0, device=0, dtype=0, wtype=0, eps=1e-5, relu=0, reserved=0)
    v.update(kw)
    return ops.NORM_ARGS.pack(*v.values())


def pack_drop(**kw):
    v = dict(M=4, N=8, x=4096, ldx=8, y=4096, ldy=8, p=0.5, seed=1, step=0, row_offset=0, state=0, stream=0, device=0, dtype=0)
    v.update(kw)
    return ops.DROPOUT_ARGS.pack(*v.values())


def pack_emb(**kw):
    v = dict(T=4, N=8, V=3, ids=4096, table=4096, ldt=8, add=0, ldadd=8, y=4096, ldy=8, dy=4096, lddy=8, dtable=4096, ws=4096,
             ws_bytes=1 << 30, stream=0, device=0, dtype=0, ids64=1, scale=1.0)
    v.update(kw)
    return ops.EMBEDDING_ARGS.pack(*v.values())


def test_packed_structs_match_the_header(tmp_path):
    """Every member of the C structs lies where struct.pack puts it: distinct values written in Python, read in C."""
    src = open(mmvae_amd.HEADER_PATH).read()
    lines = []
    for name in ("norm", "dropout", "embedding"):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct mmvae_%s_args \{(.*?)\} mmvae_%s_args;" % (name, name), src, re.S).group(1), flags=re.S)
        lines.append('printf("%s %%zu", sizeof(mmvae_%s_args));' % (name, name))
        for decl in body.split(";"):
            for member in decl.split(","):
                if member.strip():
                    m = member.split()[-1].strip("*")
                    lines.append('printf(" %%zu", offsetof(mmvae_%s_args, %s));' % (name, m))
        lines.append('printf("\\n");')
    c = tmp_path / "o.c"
    c.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"mmvae_capi.h\"\nint main(void) {%s return 0; }\n" % "\n".join(lines))
    subprocess.run(["gcc", "-I", INCLUDE, str(c), "-o", str(tmp_path / "o")], check=True)
    out = subprocess.run([str(tmp_path / "o")], check=True, capture_output=True, text=True).stdout.splitlines()
    for line, st in zip(out, (ops.NORM_ARGS, ops.DROPOUT_ARGS, ops.EMBEDDING_ARGS)):
        size, *offs = [int(v) for v in line.split()[1:]]
        assert size >= st.size and size - st.size < 8, line
        want, at = [], 0
        for n, code in re.findall(r"(\d*)([a-zA-Z])", st.format[1:]):
            for _ in range(int(n or 1)):
                want.append(at)
                at += {"q": 8, "Q": 8, "d": 8, "i": 4, "f": 4}[code]
        assert offs == want, line


NORM_BAD = [dict(M=-1), dict(N=0), dict(M=2 ** 31), dict(N=2 ** 31), dict(dtype=3), dict(wtype=1), dict(dtype=1, wtype=2), dict(eps=-1e-6),
            dict(eps=float("nan")), dict(eps=float("inf")), dict(p=-0.1), dict(p=1.1), dict(p=float("nan")), dict(x=0), dict(ldx=-1), dict(x=4098), dict(w=4097, dtype=1, wtype=1), dict(state=4100)]


@pytest.mark.parametrize("kw", NORM_BAD + [dict(y=0), dict(ldy=7), dict(y=4099, dtype=2), dict(mean=4098)])
def test_norm_forward_refuses(kw):
    L = mmvae_amd.lib()
    assert L.mmvae_layer_norm_fwd(pack_norm(**kw)) == -1
    assert L.mmvae_last_error(None).startswith(b"layer_norm_fwd: ")


@pytest.mark.parametrize("kw", NORM_BAD + [dict(dy=0), dict(mean=0), dict(rstd=0), dict(lddx=7), dict(M=5000, ws=0),
                                            dict(M=5000, ws_bytes=8), dict(lddy=-8), dict(M=1, N=2 ** 26)])
def test_norm_backward_refuses(kw):
    assert mmvae_amd.lib().mmvae_layer_norm_bwd(pack_norm(**kw)) == -1


@pytest.mark.parametrize("N", [2 ** 26 - 15, 2 ** 26 - 8, 2 ** 26 - 7, 2 ** 26 - 1, 2 ** 26])
@pytest.mark.parametrize("kw", [dict(M=0), dict(M=1), dict(M=600, ldx=0, lddy=0, dx=0), dict(db=0), dict(dw=0)])
def test_norm_backward_refuses_widths_whose_padded_sums_pass_the_grid(N, kw):
    """The weight gradients' last launch has 1024 threads for 32 of the sums of twice the width, padded to 8: 2^32 from
    N = 2^26 - 15 on."""
    L = mmvae_amd.lib()
    assert L.mmvae_layer_norm_bwd(pack_norm(N=N, lddx=N, ws_bytes=1 << 50, **kw)) == -1
    assert b"2^26 - 16" in L.mmvae_last_error(None)


@pytest.mark.parametrize("kw", [dict(M=-1), dict(N=-1), dict(N=2 ** 31), dict(dtype=5), dict(p=-1.0), dict(p=2.0), dict(p=float("nan")), dict(x=0),
                                dict(y=0), dict(ldx=-8), dict(ldy=7), dict(N=1 << 24, ldx=1 << 24, ldy=1 << 24), dict(x=4097, dtype=1),
                                dict(M=1 << 20, N=1 << 18, ldy=1 << 18)])
def test_dropout_refuses(kw):
    assert mmvae_amd.lib().mmvae_dropout(pack_drop(**kw)) == -1


@pytest.mark.parametrize("kw", [dict(T=-1), dict(N=0), dict(N=1 << 24), dict(V=-1), dict(V=2 ** 31), dict(T=2 ** 31), dict(dtype=-1), dict(ids=0),
                                dict(table=0), dict(y=0), dict(ldt=-1), dict(ldadd=-1), dict(ldy=7), dict(ids=4100), dict(table=4098),
                                dict(T=1 << 20, N=1 << 18, ldy=1 << 18)])
def test_embedding_forward_refuses(kw):
    assert mmvae_amd.lib().mmvae_embedding_fwd(pack_emb(**kw)) == -1


@pytest.mark.parametrize("kw", [dict(T=-1), dict(N=0), dict(V=-1), dict(dtype=3), dict(ids=0), dict(dy=0), dict(dtable=0), dict(dtable=4098), dict(lddy=-1),
                                dict(ws=0), dict(ws_bytes=100), dict(ws=4100), dict(V=1000, ws_bytes=100)])
def test_embedding_backward_refuses(kw):
    assert mmvae_amd.lib().mmvae_embedding_bwd(pack_emb(**kw)) == -1


def test_null_arguments_refused():
    L = mmvae_amd.lib()
    for f in ("mmvae_layer_norm_fwd", "mmvae_layer_norm_bwd", "mmvae_dropout", "mmvae_embedding_fwd", "mmvae_embedding_bwd"):
        assert getattr(L, f)(None) == -1


def test_workspace_sizes_grow_with_the_call():
    L = mmvae_amd.lib()
    assert L.mmvae_layer_norm_bwd_ws(-1, 8) == 0 and L.mmvae_layer_norm_bwd_ws(4, 0) == 0
    assert L.mmvae_embedding_bwd_ws(-1, 8, 5) == 0 and L.mmvae_embedding_bwd_ws(4, 0, 5) == 0 and L.mmvae_embedding_bwd_ws(4, 8, -1) == 0
    for N in (1, 7, 64, 100, 1000, 20000, 32768, 32769, 100000):
        for M in (0, 1, 2, 100, 2048, 4096):  # few rows: columns summed in strips, no partial sums
            n = L.mmvae_layer_norm_bwd_ws(M, N)
            assert n >= 2 * 4 * N or (n == 0 and (M <= 512 or M <= 2048 and M * N <= 1 << 22))
        assert L.mmvae_layer_norm_bwd_ws(4096, N) > 0
    # the sorted tokens (id, place), and a partial head and tail of a piece at least
    for T in (1, 4096, 4097, 600000):
        assert L.mmvae_embedding_bwd_ws(T, 33, 1000) >= 8 * T + 2 * 4 * 40
        assert L.mmvae_embedding_bwd_ws(T, 33, 7) >= 7 * 4 * 40  # few rows: a partial of each


def sums_as_the_kernels(d, gb, tg, few):
    """One id's tokens in the kernels' order and in float32: groups, pieces, shares of the pieces."""
    d = d.numpy().reshape(-1, gb, tg)
    g = np.zeros(d.shape[:2], np.float32)
    for k in range(tg):
        g += d[:, :, k]
    p = np.zeros(len(g), np.float32)
    for k in range(gb):
        p += g[:, k]
    first, rest = (np.float32(0), p) if few else (p[0], p[1:])
    shares = np.zeros(gb, np.float32)
    for j, v in enumerate(rest):
        shares[j % gb] += v
    for v in shares:
        first = np.float32(first + v)
    return float(first)


@pytest.mark.parametrize("T,N,V,gb,tg", [(262144, 136, 300, 8, 16), (262144, 256, 12, 8, 64), (262144, 600, 2, 8, 64), (1 << 20, 256, 70, 8, 16),
                                         (32768, 136, 70, 8, 8), (262144, 128, 70, 16, 16)])
def test_oracle_embedding_bound_holds_for_the_longest_chains(T, N, V, gb, tg):
    """Sums in the kernels' order that lose nearly half a step with every addition of one chain stay within the bound."""
    d = layers.longest_chain(T, gb, tg, V <= 64)
    want, bound = layers.embedding_grad(d[:, None].double().expand(T, N), torch.ones(T, dtype=torch.int64), V, 1.0)
    off = abs(sums_as_the_kernels(d, gb, tg, V <= 64) - float(want[1, 0]))
    assert off <= float(bound[1, 0]), (off / layers.U32, float(bound[1, 0]) / layers.U32)
    assert off >= 0.9 * float(bound[1, 0]) - (2 * gb + tg) * layers.U32  # (the bound is no larger than such sums need)


@pytest.mark.parametrize("M", [20000, 65536, 1 << 20])
def test_oracle_column_bound_holds_for_rows_in_sweeps(M):
    """A stripe takes every 128th row: 1 and addends just below half a step of it, each lost."""
    s = np.float32(1)
    for _ in range(M // 128 - 1):
        s += np.float32(0.999 * layers.U32)
    off = (M // 128 - 1) * 0.999 * layers.U32 + 1 - float(s)
    assert off <= layers.column_chain(M, 40000) * layers.U32
    assert M < 65536 or off > layers.column_chain(M, 20000) * layers.U32  # (those of other rows are shorter)


@pytest.mark.parametrize("N", [1, 24, 64, 128, 136, 517, 1025])  # 8, 16 and 32 lanes a row
@pytest.mark.parametrize("V", [1, 5, 12, 64, 65, 300, 30000])
def test_embedding_workspace_covers_every_smaller_call(V, N):
    """A workspace of the largest batch's size serves every smaller one (the engine keeps one): the size never falls
    as the tokens grow, over the limits of one-workgroup sorts, of long inputs and of many tiles."""
    L = mmvae_amd.lib()
    T = sorted({max(1, c + d) for c in (0, 64, 512, 4096, 20000, 32768, 33024, 40000, 65536, 262144, 524288, 1 << 20) for d in (-1, 0, 1, 64)})
    size = [L.mmvae_embedding_bwd_ws(t, N, V) for t in T]
    assert all(a <= b for a, b in zip(size, size[1:])), [(t, n) for t, n in zip(T, size)]


@pytest.mark.parametrize("N", [1, 64, 512, 1024, 2048, 2049, 3520, 3521, 4096, 4097, 20000, 20481, 32768, 32769])
def test_norm_workspace_covers_every_smaller_call(N):
    L = mmvae_amd.lib()
    size = [L.mmvae_layer_norm_bwd_ws(M, N) for M in [*range(0, 2200), 4096, 4097, 8192, 16384, 16385, 20000, 100000, 1 << 20]]
    assert all(a <= b for a, b in zip(size, size[1:]))


@pytest.mark.parametrize("call", [
    lambda t: ops.layer_norm(t),
    lambda t: ops.layer_norm_backward(t, t, t, t),
    lambda t: ops.dropout(t, 0.5, 1),
    lambda t: ops.embedding(torch.zeros(2, dtype=torch.int64), t),
    lambda t: ops.embedding_backward(t, torch.zeros(2, dtype=torch.int64), 3),
])
def test_cpu_tensors_refused(call):
    with pytest.raises(mmvae_amd.MMVAEError, match="CUDA"):
        call(torch.zeros(2, 4))


@pytest.mark.parametrize("relu", [False, True])
def test_oracle_gradients_against_differences(relu):
    """The formulas' gradients against central differences of the 64-bit forward (h = 1e-6: truncation and
    rounding both below 1e-8 of values of order 1)."""
    rng = np.random.default_rng(5)
    M, N, eps, p, seed = 5, 11, 1e-5, 0.3, 77
    x, dy = (torch.from_numpy(rng.normal(size=(M, N))) for _ in range(2))
    w, b = torch.from_numpy(1 + 0.2 * rng.normal(size=N)), torch.from_numpy(0.2 * rng.normal(size=N))
    f = layers.drop_factor(M, N, p, seed)
    u = layers.norm(x, w, b, eps, f, relu)[3]
    mask = (u > 0).double() if relu else torch.ones_like(u)
    assert u.abs().min() > 1e-3  # (no element near the ReLU's corner for the differences)
    dx, dw, db = layers.norm_grads(dy, x, w, eps, f, mask)[:3]

    def loss(x, w, b):
        return float((layers.norm(x, w, b, eps, f, relu)[0] * dy).sum())
    h = 1e-6
    for t, g, k in ((x, dx, 0), (w, dw, 1), (b, db, 2)):
        for i in np.ndindex(*t.shape):
            a = [x, w, b]
            lo, hi = t.clone(), t.clone()
            lo[i] -= h
            hi[i] += h
            a[k] = hi
            up = loss(*a)
            a[k] = lo
            assert abs((up - loss(*a)) / (2 * h) - float(g[i])) < 1e-7


def test_oracle_embedding_gradient_against_differences():
    rng = np.random.default_rng(6)
    ids = torch.tensor([2, 0, 2, -1, 5, 1, 2])  # 5: outside the table's 5 rows
    table, dy = torch.from_numpy(rng.normal(size=(5, 3))), torch.from_numpy(rng.normal(size=(7, 3)))
    g, _ = layers.embedding_grad(dy, ids, 5, 1.7)
    h = 1e-6
    for i in np.ndindex(5, 3):
        hi, lo = table.clone(), table.clone()
        hi[i] += h
        lo[i] -= h
        d = float(((layers.embedding(ids, hi, 1.7) - layers.embedding(ids, lo, 1.7)) * dy).sum()) / (2 * h)
        assert abs(d - float(g[i])) < 1e-8


@pytest.mark.parametrize("p", [0.0, 1e-6, 0.1, 0.5, 0.9, 1.0])
def test_dropout_rate_and_independence(p):
    """The kept share is 1 - thr / 65536 within 5 standard deviations; other seeds, steps and rows draw other masks."""
    M, N = 200, 1000
    k = layers.drop_kept(M, N, p, 123, 4)
    q = 1 - layers.drop_threshold(p) / 65536
    assert abs(float(k.double().mean()) - q) <= 5 * np.sqrt(q * (1 - q) / (M * N)) + 1e-12
    assert abs(q * layers.drop_scale(p) - (1 if q > 0 else 0)) < 1e-12  # the mean is kept
    if 0.05 < p < 0.95:
        for other in (layers.drop_kept(M, N, p, 124, 4), layers.drop_kept(M, N, p, 123, 5), layers.drop_kept(M, N, p, 123 + 2 ** 32, 4),
                      layers.drop_kept(M, N, p, 123, 4 + 2 ** 32)):
            agree = float((k == other).double().mean())
            assert abs(agree - (q * q + (1 - q) ** 2)) < 0.02
    # a shard's rows are the whole batch's
    assert torch.equal(layers.drop_kept(50, N, p, 123, 4, row_offset=100), k[100:150])


@pytest.mark.parametrize("kw,msg", [(dict(dropout=-0.1), "dropout"), (dict(dropout=1.0), "dropout"), (dict(dropout=float("nan")), "dropout"),
                                    (dict(n_labels=-1), "n_labels"), (dict(n_labels=2 ** 31), "n_labels"), (dict(n_labels=2, label_scale=float("inf")), "label_scale"),
                                    (dict(layer_norm=True, relu=True, enc_hidden=(8,)), "mu_encoding_1")])
def test_engine_layer_options_refused(kw, msg):
    with pytest.raises(mmvae_amd.MMVAEError, match=msg):
        mmvae_amd.Engine(D=10, K=4, **kw)


def test_label_files(tmp_path):
    f = tmp_path / "l.txt"
    f.write_text("0\n 3 \nNA\n-1\n1")
    lab, n = host.labels_read(f, 5)
    assert lab.tolist() == [0, 3, -1, -1, 1] and n == 4
    g = tmp_path / "l.gz"
    g.write_bytes(gzip.compress(b"7\n" * 5))
    assert host.labels_read(g, 5)[1] == 8
    for text, msg in (("0\n1\n", "2 labels for 5"), ("0\n" * 6, "more lines"), ("0\n\n1\n1\n1\n", "line 2"), ("0\nx\n1\n1\n1\n", "line 2"), ("1.5\n", "line 1"),
                      ("-2\n", "line 1"), ("9999999999\n", "line 1"), ("NA\n" * 5, "no cell"), ("", "0 labels")):
        f.write_text(text)
        with pytest.raises(mmvae_amd.MMVAEError, match=msg):
            host.labels_read(f, 5)
    g.write_bytes(gzip.compress(b"7\n" * 50000)[:-20])  # cut off
    with pytest.raises(mmvae_amd.MMVAEError):
        host.labels_read(g, 50000)
    with pytest.raises(mmvae_amd.MMVAEError, match="cannot read"):
        host.labels_read(tmp_path / "none", 5)


@pytest.mark.parametrize("exe", ["nb_vae_main", "vmf_vae_main"])
def test_cli_layer_options_refused(tmp_path, exe):
    p = tmp_path / "x.mtx"
    p.write_text("%%MatrixMarket matrix coordinate integer general\n3 2 2\n1 1 4\n3 2 1\n")
    lab = tmp_path / "l.txt"
    lab.write_text("0\n")
    base = [os.path.join(host.BIN_DIR, exe), "--mtx", str(p), "--out", str(tmp_path / "o")]
    for more, msg in ((["--dropout", "1.0"], "--dropout"), (["--dropout", "much"], "--dropout"), (["--label_scale", "inf"], "--label_scale"),
                      (["--labels", str(lab)], "1 labels for 2"), (["--labels", str(tmp_path / "none")], "cannot read")):
        r = subprocess.run(base + more, capture_output=True, text=True, timeout=60)
        assert r.returncode == 1 and msg in r.stderr, (more, r.stderr)


PARSE = r"""
#include <cstdio>
#include "cli.hh"
using namespace mmvae_host;
int main(int argc, const char** argv) {
    CliOptions o;
    const int rc = parse_options(argc, argv, argv[1][0] - '0', o);
    std::printf("%d %g %g %lld %lld %lld %lld %zu %s\n", rc, o.label_scale, o.dropout, (long long)o.H, (long long)o.R, (long long)o.latent,
                (long long)o.train.max_epoch, o.enc_layers.size(), o.labels.c_str());
    return 0;
}
"""


@pytest.mark.parametrize("model", ["0", "1"])
def test_cli_negative_label_scale_is_no_short_option(tmp_path, model):
    """A negative scale with an exponent reads as a scale, and nothing of it as another group's short options."""
    src, exe, lib = tmp_path / "p.cc", tmp_path / "p", os.path.dirname(mmvae_amd.LIB_PATH)
    src.write_text(PARSE)
    subprocess.run(["g++", "-std=c++17", str(src), "-o", str(exe), "-I", os.path.join(lib, "..", "host"), "-L" + lib, "-lmmvae_host", "-lmmvae",
                    "-Wl,-rpath," + lib], check=True)
    x = tmp_path / "x.mtx"
    x.write_text("")

    def parsed(*more):
        r = subprocess.run([str(exe), model, "--mtx", str(x), "--out", "o", *more], capture_output=True, text=True, check=True).stdout.split()
        return r[:2], r[2:]
    base = parsed("--labels", "f")
    assert base[0] == ["0", "1"]
    for v in ("-1e2", "-1E2", "-0.5", "-2e-3", "-1e+1", "3"):
        for name in ("--label_scale", "--label_sc"):
            for words in ((name, v), (f"{name}={v}",)):
                rc, rest = parsed(*words, "--labels", "f")
                assert rc == ["0", f"{float(v):g}"] and rest == base[1], (words, rc, rest)
    assert parsed("--label_scale")[0] == ["0", "1"]  # (no value: ignored, as all options are)
