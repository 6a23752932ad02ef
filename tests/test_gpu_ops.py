"""The layer operators (mmvae_amd.ops) against their 64-bit formulas (oracle/layers.py): sizes from one
row and one column to rows past the registers, odd widths and strides, each type, masks and ids that leave
nothing, one pass after another, captured and replayed.

Tolerances: half a step of the output's type relative to its value, plus the bound of the 32-bit
evaluation that oracle/layers.py derives from the lengths of the sums."""
import numpy as np
import pytest
import torch

import mmvae_amd
from mmvae_amd import ops
from oracle import layers

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def cpu64(t):
    return t.detach().double().cpu()


def close(got, want, bound, what):
    """|got - want| <= half a step of got's type (of the larger of the two) + bound, everywhere; equal infinities and NaN."""
    g = cpu64(got)
    assert g.shape == want.shape, (what, g.shape, want.shape)
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps  # (below the normal range: one step)
    tol = layers.half_step(got.dtype) * torch.maximum(g.abs(), want.abs()) + bound + tiny
    bad = ~((g - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((g - want).abs()[bad].max()), float(((g - want).abs() / tol)[bad].max()))


def c_norm(name, x, w, b, y=0, ldy=0, mean=0, rstd=0, dy=0, lddy=0, dx=0, lddx=0, dw=0, db=0, ws=0, ws_bytes=0):
    """The C entry itself, for outputs where the caller wants them."""
    rc = getattr(mmvae_amd.lib(), name)(ops.NORM_ARGS.pack(
        x.shape[0], x.shape[1], x.data_ptr(), x.stride(0), w.data_ptr(), b.data_ptr(), y, ldy, mean, rstd, dy, lddy, dx, lddx, dw, db, ws, ws_bytes,
        0.0, 0, 0, 0, 0, torch.cuda.current_stream().cuda_stream, 0, {F32: 0, BF16: 1, F16: 2}[x.dtype], 0, 1e-5, 0, 0))
    assert rc == 0


def make(M, N, dtype, wtype=None, pad=0, seed=0, ldy_pad=0):
    g = torch.Generator().manual_seed(1000 * M + N + seed)
    x = torch.randn(M, N + pad, generator=g) * (0.5 + torch.rand(M, 1, generator=g)) + torch.randn(M, 1, generator=g)
    x = x.to(dtype).to(DEV)[:, :N]
    dy = torch.randn(M, N + ldy_pad, generator=g).to(dtype).to(DEV)[:, :N]
    wtype = wtype or F32
    w = (1 + 0.2 * torch.randn(N, generator=g)).to(wtype).to(DEV)
    b = (0.2 * torch.randn(N, generator=g)).to(wtype).to(DEV)
    return x, dy, w, b


def check_norm(x, dy, w, b, relu=False, p=0.0, seed=0, step=0, row_offset=0, eps=1e-5, state=None, **more):
    """Forward and backward of the same call against the formulas."""
    M, N = x.shape
    kw = dict(relu=relu, p=p, seed=seed, step=step, row_offset=row_offset, state=state)
    y, mean, rstd = ops.layer_norm_forward(x, w, b, eps, **kw)
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w, b, **kw)
    one, zero = torch.ones(N).double(), torch.zeros(N).double()
    X, DY = cpu64(x), cpu64(dy)
    W, B = (cpu64(w) if w is not None else one), (cpu64(b) if b is not None else zero)
    off = [0, 0] if state is None else state.tolist()
    f = layers.drop_factor(M, N, p, seed, step + off[0], row_offset + off[1])
    Y, MEAN, RSTD, U = layers.norm(X, W, B, eps, f, relu)
    bound = layers.norm_bound(X, W, B, eps, f)
    close(y, Y, bound, "y")
    close(mean, MEAN, layers.ROW * layers.U32 * X.abs().mean(1), "mean")
    # the variance's relative error is twice a difference's, its root's half of that
    a = (RSTD[:, None] * X.abs().mean(1, keepdim=True) + 1).square()[:, 0]
    close(rstd, RSTD, 2 * layers.ROW * layers.U32 * RSTD * a, "rstd")
    mask = torch.ones(M, N).double()
    if relu:  # at the corner (|u| within its bound) either side is right: the kernel's own side, seen where y is not dropped
        mask = torch.where((U.abs() <= layers.norm_bound(X, W, B, eps, 1.0)) & (f > 0), (cpu64(y) > 0).double(), (U > 0).double())
    DX, DW, DB, bdx, bdw, bdb = layers.norm_grads(DY, X, W, eps, f, mask)
    close(dx, DX, bdx, "dx")
    close(dw, DW, bdw, "dw")
    close(db, DB, bdb, "db")
    return y, dx, dw, db


SIZES = [(1, 1), (3, 2), (5, 7), (2, 8), (33, 9), (100, 48), (64, 64), (17, 65), (70, 128), (31, 130), (9, 256), (11, 257), (5, 512), (6, 513),
         (7, 1001), (3, 1024), (3, 1025), (2, 2048), (3, 2049), (2, 4096), (2, 4097), (3, 8192), (2, 8200), (2, 12288), (2, 12296), (2, 16384), (2, 16392), (2, 20480),
         (3, 20000), (2, 20481), (2, 24576), (2, 24577), (1, 30000), (2, 32768), (2, 32769), (3, 40003)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N", SIZES)
def test_norm_sizes(M, N, dtype):
    check_norm(*make(M, N, dtype))


@pytest.mark.parametrize("relu,p", [(True, 0.0), (False, 0.3), (True, 0.3)])
@pytest.mark.parametrize("M,N", [(5, 7), (100, 48), (31, 130), (6, 513), (7, 1001), (3, 2049), (2, 8200), (2, 12296), (2, 16400), (2, 20001),
                                 (3, 20488), (1, 25000), (3, 30001), (2, 40003)])
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_relu_dropout(M, N, dtype, relu, p):
    check_norm(*make(M, N, dtype), relu=relu, p=p, seed=2 ** 40 + 99, step=2 ** 33 + 5, row_offset=1000)


@pytest.mark.parametrize("dtype,wtype", [(BF16, BF16), (F16, F16), (F32, F32), (BF16, F32)])
def test_norm_weight_types(dtype, wtype):
    x, dy, w, b = make(300, 200, dtype, wtype)
    _, _, dw, db = check_norm(x, dy, w, b)
    assert dw.dtype == wtype and db.dtype == wtype
    check_norm(x, dy, None, None)
    check_norm(x, dy, w, None)
    check_norm(x, dy, None, b, relu=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,pad,pad2", [(50, 100, 3, 0), (50, 101, 1, 5), (4, 2500, 9, 1), (2, 33000, 1, 3)])
def test_norm_strided_rows(M, N, pad, pad2, dtype):
    x, dy, w, b = make(M, N, dtype, pad=pad, ldy_pad=pad2)
    assert not x.is_contiguous()
    check_norm(x, dy, w, b, p=0.2, seed=3)


def test_norm_other_layouts():
    """Transposed and expanded inputs (repeated rows: stride 0), three dimensions, offsets into a buffer."""
    x, dy, w, b = make(64, 96, F32)
    a = ops.layer_norm_forward(x.t().contiguous().t(), w, b)[0]  # column stride not 1: copied
    assert torch.equal(a, ops.layer_norm_forward(x, w, b)[0])
    check_norm(x[:1].expand(64, 96), dy, w, b)
    check_norm(x, dy[3:4].expand(64, 96), w, b)
    y3 = ops.layer_norm_forward(x.view(4, 16, 96), w, b)
    assert y3[0].shape == (4, 16, 96) and y3[1].shape == (4, 16) and torch.equal(y3[0].view(64, 96), a)
    buf = torch.randn(64 * 96 + 1, device=DEV).to(BF16)
    check_norm(buf[1:].view(64, 96), dy.to(BF16), w, b)
    z = torch.complex(x, x).conj().imag  # lazily negated
    assert z.is_neg() and torch.equal(ops.layer_norm_forward(z, w, b)[0], ops.layer_norm_forward(-x, w, b)[0])
    v = ops.layer_norm_forward(x[0], w, b)
    assert v[0].shape == (96,) and torch.equal(v[0], a[0])


@pytest.mark.parametrize("M,N", [(4096, 128), (5000, 48), (20000, 9), (1500, 1024), (700, 20000)])
def test_norm_many_rows(M, N):
    check_norm(*make(M, N, F32), p=0.1, seed=5)
    check_norm(*make(M, N, BF16))


@pytest.mark.parametrize("p", [1.0, 0.99, 1e-7])
def test_norm_dropout_of_all_and_none(p):
    x, dy, w, b = make(60, 70, F32)
    y, dx, dw, db = check_norm(x, dy, w, b, p=p, seed=4, relu=True)
    if p == 1.0:
        assert not y.any() and not dx.any() and not dw.any() and not db.any()
        x[3, 3] = float("inf")  # (its row is dropped whole)
        y, m, r = ops.layer_norm_forward(x, w, b, p=p, seed=4)
        assert not y.any()
    if p == 1e-7:  # rounds to no dropout
        assert torch.equal(y, ops.layer_norm_forward(x, w, b, relu=True)[0])


def test_norm_offset_rows():
    """A mean far above the spread (the variance from the differences, not from squares), constant rows, zero rows."""
    x, dy, w, b = make(40, 500, F32)
    check_norm(x + 1000.0, dy, w, b)
    x[3] = 7.25
    x[4] = 0
    y, dx, _, _ = check_norm(x, dy, w, b)
    assert torch.equal(y[4], b) and torch.isfinite(dx).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("off", [0.0, 300.0, -20000.0])
@pytest.mark.parametrize("M,N", [(300, 48), (2500, 128), (40, 500), (600, 1000), (700, 2049), (1100, 4096), (600, 5000), (60, 16400), (40, 20488), (600, 33000)])
def test_norm_relu_takes_one_side_in_both_directions(M, N, off, dtype):
    """With dy = 1 the bias's gradient counts the rows whose y is above 0: the backward's u is the forward's to the bit, also
    where the mean is far above the spread and u near 0 is all rounding."""
    x, dy, w, b = make(M, N, F32)
    x = (3 * x + off).to(dtype)
    w, b = w.clamp(min=0.1), 0.01 * b
    y, mean, rstd = ops.layer_norm_forward(x, w, b, relu=True)
    _, _, db = ops.layer_norm_backward(torch.ones_like(x), x, mean, rstd, w, b, relu=True, need=(False, False, True))
    more = cpu64(db - (y > 0).sum(0))
    if dtype == F16:  # (u up to 2^-25 rounds to 0: as many rows more as have such a u within its error)
        X, W, B = cpu64(x), cpu64(w), cpu64(b)
        near = (layers.norm(X, W, B, 1e-5, 1.0, False)[3].abs() <= layers.norm_bound(X, W, B, 1e-5, 1.0) + 2.0 ** -25) & (y == 0).cpu()
        assert (more >= 0).all() and (more <= near.sum(0)).all()
    else:
        assert not more.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [7, 48, 500, 2049, 12000, 33000])
def test_norm_of_constant_rows_is_the_bias(N, dtype):
    """Rows of one value whose sum is exact in 32 bits: the mean is that value and y the bias."""
    x = torch.tensor([1.0, -3.0, 0.5, 100.0, 0.0], device=DEV).to(dtype)[:, None].expand(5, N).contiguous()
    _, dy, w, b = make(5, N, dtype)
    y, mean, rstd = ops.layer_norm_forward(x, w, b)
    assert torch.equal(mean, x[:, 0].float()) and torch.equal(y, b.to(dtype).expand(5, N))
    check_norm(x, dy, w, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("off", [30.0, 1000.0, -5000.0])
@pytest.mark.parametrize("M,N", [(40, 500), (600, 1000), (5, 16400), (3, 33000), (2500, 96)])
def test_norm_of_rows_far_from_zero(M, N, off, dtype):
    """Means far above the spread: in 16 bits such rows hold few different values, or one."""
    x, dy, w, b = make(M, N, F32)
    x, dy = (3 * x + off).to(dtype), dy.to(dtype)
    check_norm(x, dy, w, b)
    check_norm(x, dy, w, b, relu=True, p=0.25, seed=3)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_rows_of_one_value_or_one_other(dtype):
    x, dy, w, b = make(12, 4000, dtype)
    x = x.clone()
    for r, v in enumerate((3.3, 0.0, 60000.0, 1e-6, 0.1, 100.0)):
        x[r] = v
    x[4, 7], x[5, 9] = 0.2, 101.0
    check_norm(x, dy, w, b)
    check_norm(x, dy, w, b, eps=1e-12)


def test_norm_infinities_stay_in_their_rows():
    x, dy, w, b = make(40, 500, F32)
    clean = ops.layer_norm_forward(x, w, b)
    cdx = ops.layer_norm_backward(dy, x, clean[1], clean[2], w, b, need=(True, False, False))[0]
    bad = x.clone()
    bad[7, 3], bad[9, 0] = float("nan"), float("inf")
    y, mean, rstd = ops.layer_norm_forward(bad, w, b)
    dx = ops.layer_norm_backward(dy, bad, mean, rstd, w, b, need=(True, False, False))[0]
    keep = torch.ones(40, dtype=torch.bool)
    keep[[7, 9]] = False
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], cdx[keep])
    assert torch.isnan(y[7]).all() and torch.isnan(y[9]).all() and torch.isnan(dx[7]).all()
    # a ReLU keeps a NaN
    assert torch.isnan(ops.layer_norm_forward(bad, w, b, relu=True)[0][7]).all()


def test_norm_no_rows_and_parts():
    x, dy, w, b = make(16, 64, F32)
    y, mean, rstd = ops.layer_norm_forward(x[:0], w, b)
    assert y.shape == (0, 64) and mean.shape == (0,)
    dx, dw, db = ops.layer_norm_backward(dy[:0], x[:0], mean, rstd, w, b)
    assert dx.shape == (0, 64) and not dw.any() and not db.any()
    full = ops.layer_norm_forward(x, w, b)
    all3 = ops.layer_norm_backward(dy, x, full[1], full[2], w, b)
    assert ops.layer_norm_forward(x, w, b, stats=False)[1:] == (None, None)
    for k in range(3):
        need = tuple(i == k for i in range(3))
        part = ops.layer_norm_backward(dy, x, full[1], full[2], w, b, need=need)
        assert torch.equal(part[k], all3[k]) and all(part[i] is None for i in range(3) if i != k)


def test_norm_weight_gradients_of_the_widest_rows():
    """No rows of the largest width that is taken: its last launch has the most threads, and clears both sums."""
    N = 2 ** 26 - 16
    x, st = torch.empty(0, N, device=DEV), torch.empty(0, device=DEV)
    w = torch.ones(N, device=DEV)
    dx, dw, db = ops.layer_norm_backward(x, x, st, st, w)
    assert dx.shape == (0, N) and not dw.any() and not db.any()
    with pytest.raises(mmvae_amd.MMVAEError, match="2\\^26 - 16"):
        x = torch.empty(0, N + 1, device=DEV)
        ops.layer_norm_backward(x, x, st, st)


def test_norm_equal_calls_equal_bits():
    x, dy, w, b = make(3000, 300, F32)
    one = check_norm(x, dy, w, b, p=0.2, seed=1)
    for _ in range(3):
        for a, c in zip(one, check_norm(x, dy, w, b, p=0.2, seed=1)):
            assert torch.equal(a, c)


def test_norm_in_place():
    """y over x, dx over dy: rows are read whole before they are written (also where they are read in sweeps)."""
    for M, N in ((100, 48), (5, 2049), (3, 40003)):
        x, dy, w, b = make(M, N, F32)
        x, dy = x.contiguous(), dy.contiguous()
        y, mean, rstd = ops.layer_norm_forward(x, w, b)
        dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w, b)
        dy2, dw2, db2 = dy.clone(), torch.empty_like(dw), torch.empty_like(db)
        n = mmvae_amd.lib().mmvae_layer_norm_bwd_ws(M, N)
        ws = torch.empty(n, dtype=torch.uint8, device=DEV)
        c_norm("mmvae_layer_norm_bwd", x, w, b, mean=mean.data_ptr(), rstd=rstd.data_ptr(), dy=dy2.data_ptr(), lddy=N, dx=dy2.data_ptr(), lddx=N,
               dw=dw2.data_ptr(), db=db2.data_ptr(), ws=ws.data_ptr(), ws_bytes=n)
        assert torch.equal(dy2, dx) and torch.equal(dw2, dw) and torch.equal(db2, db)
        c_norm("mmvae_layer_norm_fwd", x, w, b, y=x.data_ptr(), ldy=N)
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N", [(2048, 9), (2049, 9), (513, 64), (1025, 129), (2048, 2048), (2048, 2049), (1023, 4097), (204, 20480), (512, 4097), (513, 4097), (129, 8193), (70, 20481), (3, 33001), (1200, 3520), (1200, 3521), (1100, 4096)])
def test_norm_gradients_in_strips_and_in_parts(M, N, dtype):
    """Both sides of the limits up to which a backward sums its columns in strips beside the rows."""
    x, dy, w, b = make(M, N, dtype)
    check_norm(x, dy, w, b)
    check_norm(x, dy, w, b, relu=True, p=0.3, seed=5, step=9)


@pytest.mark.parametrize("M,N", [(1, 7), (100, 129), (700, 1024), (3, 9000), (300, 5000), (2500, 500), (600, 5000), (40, 21001)])
@pytest.mark.parametrize("over", ["dy", "x"])
def test_norm_backward_over_its_inputs(M, N, over):
    x, dy, w, b = make(M, N, BF16)
    x, dy = x.contiguous(), dy.contiguous()
    _, mean, rstd = ops.layer_norm_forward(x, w, b)
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w, b)
    x2, dy2, dw2, db2 = x.clone(), dy.clone(), torch.empty_like(dw), torch.empty_like(db)
    out = dy2 if over == "dy" else x2
    n = mmvae_amd.lib().mmvae_layer_norm_bwd_ws(M, N)
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    c_norm("mmvae_layer_norm_bwd", x2, w, b, mean=mean.data_ptr(), rstd=rstd.data_ptr(), dy=dy2.data_ptr(), lddy=N, dx=out.data_ptr(), lddx=N,
           dw=dw2.data_ptr(), db=db2.data_ptr(), ws=ws.data_ptr() if n else 0, ws_bytes=n)
    assert torch.equal(out, dx) and torch.equal(dw2, dw) and torch.equal(db2, db)


@pytest.mark.parametrize("dtype,N,masked", [(BF16, 20000, False), (F16, 16400, False), (BF16, 30000, False), (F32, 20000, False),
                                            (BF16, 12296, True), (F16, 20000, True), (F32, 8200, True)])
def test_norm_backward_after_one_that_left_nan_in_lds(dtype, N, masked):
    """Rows whose weights lie in LDS and whose last chunks leave lanes idle: what such a lane multiplies its zeros with is
    not what an earlier call (here one with weights of NaN, on every CU) left there."""
    x, dy, w, b = make(700, N, dtype)
    kw = dict(p=0.2, seed=3) if masked else {}
    _, mean, rstd = ops.layer_norm_forward(x, w, b, **kw)
    nan = torch.full_like(w, float("nan"))
    want = None
    for _ in range(4):
        assert torch.isnan(ops.layer_norm_backward(dy, x, mean, rstd, nan, b, **kw)[0]).all()
        got = ops.layer_norm_backward(dy, x, mean, rstd, w, b, **kw)
        assert all(torch.isfinite(t).all() for t in got)
        assert want is None or all(torch.equal(t, u) for t, u in zip(got, want))
        want = got
    check_norm(x[:3], dy[:3], w, b, **kw)


def test_norm_leaves_what_is_beside_its_rows():
    """Outputs with a row stride above N: the columns between the rows stay as they were."""
    M, N, ld = 37, 101, 120
    x, dy, w, b = make(M, N, BF16)
    buf = torch.full((M + 2, ld), 5.0, dtype=BF16, device=DEV)
    c_norm("mmvae_layer_norm_fwd", x, w, b, y=buf[1].data_ptr(), ldy=ld)
    assert torch.equal(buf[1:M + 1, :N], ops.layer_norm_forward(x, w, b)[0])
    assert (buf[:, N:] == 5).all() and (buf[0] == 5).all() and (buf[-1] == 5).all()


# ---- dropout ---------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,pad", [(1, 1, 0), (5, 3, 0), (100, 128, 0), (33, 129, 0), (7, 1001, 6), (300, 2500, 0), (3, 20001, 1), (70000, 5, 0)])
def test_dropout_bits(M, N, pad, dtype):
    """Every element is x times the factor in 32 bits, rounded once, or 0: equal bits."""
    x = make(M, N, dtype, pad=pad)[0]
    for p, seed, step, ro in ((0.25, 7, 0, 0), (0.9, 2 ** 63 + 11, 2 ** 40 + 1, 2 ** 32 - 2), (0.0, 1, 1, 1), (1.0, 1, 1, 1), (1e-6, 1, 1, 1)):
        y = ops.dropout_apply(x, p, seed, step=step, row_offset=ro)
        keep = layers.drop_kept(M, N, p, seed, step, ro).to(DEV)
        want = torch.where(keep, (x.float() * np.float32(layers.drop_scale(p))).to(dtype), torch.zeros((), dtype=dtype, device=DEV))
        assert y.dtype == dtype and torch.equal(y, want), (p, seed)


def test_state_changed_before_the_backward_is_refused():
    x, _, w, b = make(9, 40, F32)
    x.requires_grad_()
    state = torch.zeros(2, dtype=torch.int64, device=DEV)
    for f in (lambda: ops.dropout(x, 0.5, 3, state=state), lambda: ops.layer_norm(x, w, b, p=0.5, seed=3, state=state)):
        y = f()
        state += 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
        f().sum().backward()


def test_dropout_same_mask_as_the_norm_and_backward():
    x, dy, w, b = make(200, 77, F32)
    key = dict(p=0.4, seed=1234, step=9, row_offset=3)
    kept = ops.dropout_apply(torch.ones_like(x), 0.4, 1234, step=9, row_offset=3) != 0
    plain = ops.layer_norm_forward(x, w, b)[0]
    y = ops.layer_norm_forward(x, w, b, **key)[0]
    s = np.float32(layers.drop_scale(0.4))
    assert torch.equal(y != 0, kept & (plain != 0))
    # xh (w s) + b s in place of (xh w + b) s: four roundings of values up to (|xh w| + |b|) s
    tol = 4 * layers.U32 * (plain.abs() + 2 * b.abs()) * float(s)
    assert ((y - torch.where(kept, plain * s, torch.zeros_like(x))).abs() <= tol).all()
    a = x.clone().requires_grad_()
    ops.dropout(a, 0.4, 1234, step=9, row_offset=3).backward(dy)
    assert torch.equal(a.grad, torch.where(kept, dy * s, torch.zeros_like(x)))


def test_dropout_of_infinities():
    x = torch.full((50, 40), float("inf"), device=DEV)
    x[:, ::2] = float("nan")
    y = ops.dropout_apply(x, 0.5, 3)
    kept = layers.drop_kept(50, 40, 0.5, 3).to(DEV)
    assert (y[~kept] == 0).all() and not torch.isfinite(y[kept]).any()
    assert ops.dropout_apply(x[:0], 0.5, 3).shape == (0, 40)


def test_dropout_shards():
    x = make(96, 50, F32)[0]
    whole = ops.dropout_apply(x, 0.3, 5, step=2)
    parts = [ops.dropout_apply(x[r:r + 32], 0.3, 5, step=2, row_offset=r) for r in (0, 32, 64)]
    assert torch.equal(whole, torch.cat(parts))


# ---- embedding -------------------------------------------------------------------------------
def tokens(T, V, skew, seed=0, dtype=torch.int64, holes=True):
    g = torch.Generator().manual_seed(T + 7 * V + seed)
    if skew:
        ids = ((torch.rand(T, generator=g, dtype=torch.float64) * np.log(V + 1)).exp() - 1).long().clamp_(0, V - 1)
        ids = torch.randperm(V, generator=g)[ids]
    else:
        ids = torch.randint(0, V, (T,), generator=g)
    if holes and T > 8:
        ids[torch.randint(0, T, (max(1, T // 50),), generator=g)] = -1
        ids[T // 2] = V  # outside on the other side
    return ids.to(dtype).to(DEV)


def check_embedding(ids, V, N, dtype, scale=1.5, add=False, seed=0):
    g = torch.Generator().manual_seed(seed + V)
    table = torch.randn(V, N, generator=g).to(dtype).to(DEV)
    T = ids.numel()
    dy = torch.randn(*ids.shape, N, generator=g).to(dtype).to(DEV)
    extra = torch.randn(*ids.shape, N, generator=g).to(dtype).to(DEV) if add else None
    y = ops.embedding_forward(ids, table, scale, extra)
    s = float(np.float32(scale))
    # one product (and sum) in 32 bits, then the rounding
    Y = layers.embedding(ids.cpu(), cpu64(table), s, cpu64(extra) if add else None)
    close(y, Y, 2 * layers.U32 * Y.abs(), "y")
    d = ops.embedding_backward(dy, ids, V, scale)
    D, bound = layers.embedding_grad(cpu64(dy), ids.cpu(), V, s)
    close(d, D, bound, "dtable")
    assert torch.equal(d, ops.embedding_backward(dy, ids, V, scale))
    return y, d


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,N,skew", [(1, 1, 1, False), (1, 30, 64, False), (2, 1, 8, False), (7, 3, 5, False), (100, 4, 48, False), (513, 255, 65, True),
                                        (1000, 256, 128, True), (4096, 12, 128, False), (4097, 2, 130, False), (5000, 70000, 16, True),
                                        (9000, 300, 517, True), (40000, 1, 33, False), (33000, 20000, 24, True), (70000, 5, 300, False),
                                        (3000, 7, 2100, True)])
def test_embedding_sizes(T, V, N, skew, dtype):
    check_embedding(tokens(T, V, skew), V, N, dtype)


@pytest.mark.parametrize("T,V", [(600000, 50), (530000, 66000)])
def test_embedding_many_tiles(T, V):
    """More sort tiles than a scatter workgroup sums itself; two and three digits."""
    check_embedding(tokens(T, V, True), V, 9, F32)


@pytest.mark.parametrize("N,V,gb,tg", [(136, 300, 8, 16), (256, 12, 8, 64)])
def test_embedding_hot_id_of_many_tokens(N, V, gb, tg):
    """262144 tokens of one id, whose sum loses nearly half a step with each addition of its longest chain, and random ones."""
    T = 262144
    ids = torch.full((T,), V - 1, device=DEV)
    for col in (layers.longest_chain(T, gb, tg, V <= 64), torch.randn(T, generator=torch.Generator().manual_seed(N))):
        d = ops.embedding_backward(col[:, None].to(DEV).expand(T, N), ids, V)
        D, bound = layers.embedding_grad(col[:, None].double().expand(T, N), ids.cpu(), V, 1.0)
        close(d, D, bound, "dtable")


@pytest.mark.parametrize("T,V,N", [(300, 5, 40), (5000, 300, 130), (33000, 12, 24)])
@pytest.mark.parametrize("dtype", TYPES)
def test_embedding_gradient_of_strided_and_repeated_rows(T, V, N, dtype):
    """dy inside wider rows, with a column stride, transposed, one row for all tokens, one value for all."""
    g = torch.Generator().manual_seed(T)
    ids = tokens(T, V, True)
    wide = torch.randn(T, 2 * N + 3, generator=g).to(dtype).to(DEV)
    for dy in (wide[:, 3:N + 3], wide[:, 1:2 * N + 1:2], wide[:, :N].t().contiguous().t(), wide[:1, :N].expand(T, N), wide[:1, :1].expand(T, N),
               wide[:, :1].expand(T, N)):
        d = ops.embedding_backward(dy, ids, V, 0.5)
        D, bound = layers.embedding_grad(cpu64(dy), ids.cpu(), V, 0.5)
        close(d, D, bound, "dtable")
        assert torch.equal(d, ops.embedding_backward(dy.contiguous(), ids, V, 0.5))


def test_embedding_id_types_shapes_add():
    ids = tokens(600, 50, True)
    a = check_embedding(ids, 50, 40, F32, add=True)
    b = check_embedding(ids.to(torch.int32), 50, 40, F32, add=True)
    c = check_embedding(ids.view(6, 100), 50, 40, F32, add=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[0].view(6, 100, 40), c[0]) and torch.equal(a[1], c[1])
    far = torch.tensor([2 ** 40, -2 ** 40, 2 ** 32 + 1, 1], device=DEV)  # (not cut to 32 bits)
    check_embedding(far, 5, 8, F32)


def test_embedding_nothing_to_look_up():
    t = torch.randn(5, 8, device=DEV)
    none = torch.full((300,), -1, device=DEV)
    assert not ops.embedding_forward(none, t).any()
    assert not ops.embedding_backward(torch.randn(300, 8, device=DEV), none, 5).any()
    empty = none[:0]
    assert ops.embedding_forward(empty, t).shape == (0, 8)
    assert not ops.embedding_backward(torch.randn(0, 8, device=DEV), empty, 5).any()
    assert ops.embedding_backward(torch.randn(300, 8, device=DEV), none, 0).shape == (0, 8)
    assert not ops.embedding_forward(none, t[:0]).any()
    for V, N in ((1, 1), (3, 3), (1001, 1)):  # an odd number of 16-bit elements is cleared whole, and nothing behind it
        d = ops.embedding_backward(torch.randn(300, N, device=DEV).to(BF16), none, V)
        assert d.shape == (V, N) and not d.any()


def test_embedding_unlabelled_rows_do_not_spread():
    """NaN in the gradient of a token without a label reaches no row; in a labelled one only its row."""
    ids = torch.tensor([0, -1, 2, 2, 1], device=DEV)
    dy = torch.ones(5, 8, device=DEV)
    dy[1] = float("nan")
    d = ops.embedding_backward(dy, ids, 4, 2.0)
    assert torch.equal(d[:, 0].cpu(), torch.tensor([2.0, 2.0, 4.0, 0.0]))
    dy[4] = float("nan")
    d = ops.embedding_backward(dy, ids, 4, 2.0)
    assert torch.isnan(d[1]).all() and torch.isfinite(d[[0, 2, 3]]).all()


@pytest.mark.parametrize("T", [64, 255, 256, 257, 511, 512, 513, 1025, 4095, 8192, 33024])
@pytest.mark.parametrize("N", [8, 100, 600])
def test_embedding_runs_at_the_pieces_edges(T, N):
    """One id everywhere, two ids that change at every place around a piece's end, runs of one token."""
    for ids in (torch.zeros(T), (torch.arange(T) >= T // 2).float(), (torch.arange(T) >= T - 1).float(), (torch.arange(T) >= 256).float(), torch.arange(T) // 3):
        check_embedding(ids.long().to(DEV), max(2, T // 3 + 1), N, F32, seed=T)


def test_embedding_far_offsets():
    """A table and a gradient of more than 2^31 elements, rows whose stride passes 2^31."""
    V, N = 2 ** 21 + 3, 1024
    ids = torch.tensor([0, V - 1, V - 2, V - 1], device=DEV)
    table = torch.zeros(V, N, dtype=BF16, device=DEV)
    table[V - 1], table[V - 2], table[0] = 3, 2, 1
    y = ops.embedding_forward(ids, table, 2.0)
    assert torch.equal(y[:, 0].cpu().float(), torch.tensor([2.0, 6, 4, 6]))
    del table
    d = ops.embedding_backward(y, ids, V, 0.5)
    assert d[V - 1, 5] == 6 and d[V - 2, 1023] == 2 and d[0, 0] == 1
    assert int((d != 0).sum()) == 3 * N
    del d
    buf = torch.randn(2 ** 31 + 4096, dtype=BF16, device=DEV)
    x = buf.as_strided((2, 300), (2 ** 31 + 64, 1))
    w, b = torch.ones(300, device=DEV), torch.zeros(300, device=DEV)
    assert torch.equal(ops.layer_norm_forward(x, w, b)[0], ops.layer_norm_forward(x.contiguous(), w, b)[0])
    assert torch.equal(ops.dropout_apply(x, 0.5, 1), ops.dropout_apply(x.contiguous(), 0.5, 1))


# ---- together --------------------------------------------------------------------------------
def test_chain_gradients_against_autograd_in_64_bits():
    """label vector + hidden layer -> norm, ReLU, dropout -> Linear -> norm -> dropout, twice the same label table,
    gradients of every leaf (the table's from both places) against autograd of the formulas in 64 bits."""
    T, V, N, H = 300, 7, 40, 56
    g = torch.Generator().manual_seed(3)
    leaves = [torch.randn(V, N, generator=g), torch.randn(T, N, generator=g), 1 + 0.1 * torch.randn(N, generator=g), 0.1 * torch.randn(N, generator=g),
              torch.randn(H, N, generator=g) / N ** 0.5, 1 + 0.1 * torch.randn(H, generator=g), 0.1 * torch.randn(H, generator=g)]
    ids = tokens(T, V, False)
    out = torch.randn(T, H, generator=g)

    def chain(table, x, w1, b1, lin, w2, b2, norm, drop, emb):
        h = norm(emb(table, 2.0, x), w1, b1, True, 0.2, 11)
        h = norm(h @ lin.t(), w2, b2, False, 0.0, 0)
        return drop(h, 0.3, 12)
    dev = [t.to(DEV).requires_grad_() for t in leaves]
    y = chain(*dev, norm=lambda x, w, b, r, p, s: ops.layer_norm(x, w, b, relu=r, p=p, seed=s), drop=lambda x, p, s: ops.dropout(x, p, s, step=4),
              emb=lambda t, s, x: ops.embedding(ids, t, s, ops.embedding(ids, t, -0.5, x)))
    y.backward(out.to(DEV))
    ref = [t.double().requires_grad_() for t in leaves]
    i = ids.cpu()
    z = chain(*ref, norm=lambda x, w, b, r, p, s: layers.norm(x, w, b, 1e-5, layers.drop_factor(*x.shape, p, s), r)[0],
              drop=lambda x, p, s: x * layers.drop_factor(*x.shape, p, s, 4),
              emb=lambda t, s, x: layers.embedding(i, t, s, layers.embedding(i, t, -0.5, x)))
    z.backward(out.double())
    # 32-bit evaluation of a chain of some 2,000 roundings with factors of order 1: 2e-4 of the largest value
    for a, b in [(y, z)] + [(d.grad, r.grad) for d, r in zip(dev, ref)]:
        assert (cpu64(a) - b.detach()).abs().max() <= 2e-4 * b.detach().abs().max()


def test_autograd_only_where_needed():
    x, dy, w, b = make(20, 30, F32)
    w.requires_grad_()
    ops.layer_norm(x, w, b).backward(dy)
    assert w.grad is not None
    with torch.no_grad():
        assert not ops.layer_norm(x, w, b).requires_grad
    t = torch.randn(4, 8, device=DEV)
    e = torch.randn(3, 8, device=DEV, requires_grad=True)
    ops.embedding(torch.tensor([0, 1, -1], device=DEV), t, 1.0, e).backward(torch.ones(3, 8, device=DEV))
    assert torch.equal(e.grad, torch.ones(3, 8, device=DEV))
    with pytest.raises(RuntimeError):  # no second derivative
        y = ops.layer_norm(x, w, b)
        gr, = torch.autograd.grad(y.sum(), w, create_graph=True)
        gr.sum().backward()


def test_other_streams_and_threads():
    """Two streams with their own inputs at the same time, from two threads; each as alone."""
    import threading
    sets = [make(2000, 300, F32, seed=s) for s in (1, 2)]
    ids = [tokens(6000, 50, True, seed=s) for s in (1, 2)]
    dy = [torch.randn(6000, 64, device=DEV) for _ in range(2)]
    want = [(ops.layer_norm_forward(s[0], s[2], s[3], p=0.1, seed=1), ops.embedding_backward(d, i, 50)) for s, i, d in zip(sets, ids, dy)]
    want = [(w[0][0], w[1]) for w in want]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(k):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(20):
                    y = ops.layer_norm_forward(sets[k][0], sets[k][2], sets[k][3], p=0.1, seed=1)[0]
                    d = ops.embedding_backward(dy[k], ids[k], 50)
            st.synchronize()
            got[k] = (y, d)
        except Exception as e:  # (reported by the main thread)
            errors.append(e)
    th = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in th:
        t.start()
    for t in th:
        t.join()
    assert not errors
    for k in range(2):
        assert torch.equal(got[k][0], want[k][0]) and torch.equal(got[k][1], want[k][1])


def test_captured_and_replayed():
    """Forward and backward of all operators in a graph; every replay, with new inputs, ids and dropout state and eager
    work between, equals the eager calls; a second graph over the same inputs keeps its own workspace."""
    x, dy, w, b = make(500, 130, F32)
    ids, table = tokens(5000, 40, True), torch.randn(40, 130, device=DEV)
    de = torch.randn(5000, 130, device=DEV)
    state = torch.zeros(2, dtype=torch.int64, device=DEV)

    def run():
        y, m, r = ops.layer_norm_forward(x, w, b, relu=True, p=0.2, seed=9, step=1, state=state)
        g = ops.layer_norm_backward(dy, x, m, r, w, b, relu=True, p=0.2, seed=9, step=1, state=state)
        d = ops.dropout_apply(x, 0.5, 8, state=state)
        return [y, *g, d, ops.embedding_forward(ids, table, 2.0), ops.embedding_backward(de, ids, 40, 2.0)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o = run()
        graphs.append(gr)
        outs.append(o)
    for k in range(4):
        x.copy_(torch.randn_like(x))
        ids.copy_(tokens(5000, 40, k % 2 == 0, seed=k))
        de.copy_(torch.randn_like(de))
        state.copy_(torch.tensor([k, 100 * k]))
        want = [t.clone() for t in run()]
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for o in outs:
            for a, c in zip(o, want):
                assert torch.equal(a, c), k
        run()
    # the state does what step and row_offset do
    a = ops.dropout_apply(x, 0.5, 8, state=torch.tensor([3, 300], device=DEV))
    assert torch.equal(a, ops.dropout_apply(x, 0.5, 8, step=3, row_offset=300))


def test_python_refusals():
    x, dy, w, b = make(8, 16, F32)
    y, m, r = ops.layer_norm_forward(x, w, b)
    E = mmvae_amd.MMVAEError
    for call in (lambda: ops.layer_norm(x.double()), lambda: ops.layer_norm(x, w[:8]), lambda: ops.layer_norm(x, w.to(BF16)),
                 lambda: ops.layer_norm(x.to(BF16), w.to(BF16), b), lambda: ops.layer_norm(x, w.cpu()), lambda: ops.layer_norm(x, w, b, eps=-1.0),
                 lambda: ops.layer_norm(x, p=1.5), lambda: ops.layer_norm(x, w.repeat(2)[::2]), lambda: ops.layer_norm(torch.zeros((), device=DEV)),
                 lambda: ops.layer_norm(x[:, :0]), lambda: ops.layer_norm(x, state=torch.zeros(2, device=DEV)),
                 lambda: ops.layer_norm(x, state=torch.zeros(2, dtype=torch.int64)),
                 lambda: ops.layer_norm_backward(dy[:4], x, m, r, w, b), lambda: ops.layer_norm_backward(dy.to(BF16), x, m, r, w, b),
                 lambda: ops.layer_norm_backward(dy, x, m[:4], r, w, b), lambda: ops.layer_norm_backward(dy, x, m.double(), r, w, b),
                 lambda: ops.dropout(x, -0.1, 1), lambda: ops.dropout(x.int(), 0.1, 1),
                 lambda: ops.embedding(torch.zeros(3, device=DEV), x), lambda: ops.embedding(torch.zeros(3, dtype=torch.int64), x),
                 lambda: ops.embedding(torch.zeros(3, dtype=torch.int64, device=DEV), x, 1.0, x),
                 lambda: ops.embedding(torch.zeros(3, dtype=torch.int64, device=DEV), x[0]),
                 lambda: ops.embedding_backward(dy, torch.zeros(3, dtype=torch.int64, device=DEV), 4),
                 lambda: ops.embedding_backward(dy, torch.zeros(8, dtype=torch.int64, device=DEV), -1)):
        with pytest.raises(E):
            call()
    assert torch.equal(ops.layer_norm_forward(x, w, b)[0], y)
