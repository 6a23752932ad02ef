"""Layer operators on torch tensors: layer norm (with ReLU and dropout in the same pass), dropout and
embedding lookup, forward and backward (ctypes over include/mmvae_capi.h, "layer operators").

The layers around the count VAEs' Linears (the reference builds those chains at
include/models/nb.hh:331-379 and include/models/vmf.hh:338-385): the engine runs the same kernels in
its hidden layers (``Engine(layer_norm=True, dropout=0.1, n_labels=V)``); here they take CUDA tensors.

``layer_norm``, ``dropout`` and ``embedding`` are differentiable; ``*_forward`` / ``*_backward`` /
``dropout_apply`` are the bare calls, for callers with a backward pass of their own (and for capture
into a graph, where autograd's bookkeeping has no place).  All work is enqueued on the current stream
of the tensors' device.  Types: float32, bfloat16, float16; weights and biases in the same type or
float32.  Wrong arguments raise :class:`MMVAEError` before anything runs; there is no CPU path.

Dropout is a function of ``(seed, step, row, column)``: a call with the same key drops the same
elements (``Engine``'s noise is keyed alike), so nothing is stored between forward and backward, and
a data-parallel shard passes its first row as ``row_offset``.  ``state``, an int64 CUDA tensor
``[step, row_offset]`` added to the two, lets a captured graph's replays draw new masks.
"""
import struct

import torch

from . import MMVAEError, lib

_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MASK = (1 << 64) - 1
# the argument structs, member by member (8-byte members first: no padding)
_NORM = struct.Struct("=2q Q q 2Q Q q 2Q Q q Q q 2Q Q q d 3Q Q Q 3i f 2i")
_DROP = struct.Struct("=2q Q q Q q d 3Q Q Q 2i")
_EMB = struct.Struct("=3q 2Q q Q q Q q Q q Q Q q Q 3i f")


def _wrong(what):
    raise MMVAEError(what)


def _rows(t, name, like=None):
    """t as [rows, N] with unit column stride (a view where it is one); its row stride."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _wrong(f"{name} must be a CUDA tensor")
    if t.dtype not in _TYPE:
        _wrong(f"{name}: float32, bfloat16 or float16, not {t.dtype}")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        _wrong(f"{name} must have the shape, type and device of the other tensors")
    if t.dim() == 0 or t.shape[-1] == 0:
        _wrong(f"{name} needs a last dimension of at least 1")
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1 and t.shape[1] > 1:
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else t.shape[1])


def _weight(t, name, x):
    if t is None:
        return 0
    if not isinstance(t, torch.Tensor) or t.device != x.device or t.shape != (x.shape[-1],):
        _wrong(f"{name} must be a tensor of [{x.shape[-1]}] on x's device")
    if t.dtype != x.dtype and t.dtype != torch.float32:
        _wrong(f"{name}: x's type or float32, not {t.dtype}")
    if t.stride(0) != 1 and t.shape[0] > 1:
        _wrong(f"{name} must be contiguous")
    return t.data_ptr()


def _state(state, x):
    if state is None:
        return 0
    if not isinstance(state, torch.Tensor) or state.device != x.device or state.dtype != torch.int64 or state.numel() != 2 or not state.is_contiguous():
        _wrong("state must be a contiguous int64 tensor [step, row_offset] on x's device")
    return state.data_ptr()


def _stream(x):
    return torch.cuda.current_stream(x.device).cuda_stream, x.device.index


def _call(name, args):
    rc = getattr(lib(), name)(args)
    if rc != 0:
        _wrong(f"{name} failed ({rc}): {lib().mmvae_last_error(None).decode()}")


def _norm_args(x, ldx, w, b, wtype, y=0, ldy=0, mean=0, rstd=0, dy=0, lddy=0, dx=0, lddx=0, dw=0, db=0, ws=0, ws_bytes=0,
               eps=0.0, relu=False, p=0.0, seed=0, step=0, row_offset=0, state=0):
    st, dev = _stream(x)
    return _NORM.pack(x.shape[0], x.shape[1], x.data_ptr(), ldx, w, b, y, ldy, mean, rstd, dy, lddy, dx, lddx, dw, db, ws, ws_bytes,
                      p, seed & _MASK, step & _MASK, row_offset & _MASK, state, st, dev, _TYPE[x.dtype], wtype, eps, 1 if relu else 0, 0)


def _wtype(x, weight, bias):
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        _wrong("weight and bias must have one type")
    t = weight if weight is not None else bias
    return _TYPE.get(t.dtype, -1) if t is not None else 0


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, *, relu=False, p=0.0, seed=0, step=0, row_offset=0, state=None, stats=True):
    """y, mean, rstd of drop(relu?(norm(x) * weight + bias)) over x's last dimension; ``stats=False`` (serving)
    stores no statistics and returns None for them."""
    x2, ldx = _rows(x, "x")
    w, b = _weight(weight, "weight", x2), _weight(bias, "bias", x2)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    M, N = x2.shape
    mean = rstd = None
    if stats:
        both = torch.empty((2, M), dtype=torch.float32, device=x.device)
        mean, rstd = both[0], both[1]
    _call("mmvae_layer_norm_fwd", _norm_args(
        x2, ldx, w, b, _wtype(x2, weight, bias), y=y.data_ptr(), ldy=N, mean=mean.data_ptr() if stats else 0,
        rstd=rstd.data_ptr() if stats else 0, eps=eps, relu=relu, p=p, seed=seed, step=step, row_offset=row_offset,
        state=_state(state, x2)))
    if stats and x.dim() != 2:
        mean, rstd = mean.view(x.shape[:-1]), rstd.view(x.shape[:-1])
    return y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight=None, bias=None, *, relu=False, p=0.0, seed=0, step=0, row_offset=0, state=None,
                        need=(True, True, True)):
    """dx, dweight, dbias (of weight's type, float32 without one; None where ``need`` says so) from the forward's
    x and statistics; ReLU and dropout as the forward had them (its bias is needed for the ReLU)."""
    x2, ldx = _rows(x, "x")
    dy2, lddy = _rows(dy, "dy", x)
    w, b = _weight(weight, "weight", x2), _weight(bias, "bias", x2)
    M, N = x2.shape
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != x.device or t.numel() != M or not t.is_contiguous():
            _wrong(f"{name} must be the forward's float32 statistics")
    wtype = _wtype(x2, weight, bias)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
    wt = (weight if weight is not None else bias).dtype if weight is not None or bias is not None else torch.float32
    dw = torch.empty(N, dtype=wt, device=x.device) if need[1] else None
    db = torch.empty(N, dtype=wt, device=x.device) if need[2] else None
    ws, n = None, 0
    if need[1] or need[2]:
        n = lib().mmvae_layer_norm_bwd_ws(M, N)
        ws = torch.empty(n, dtype=torch.uint8, device=x.device)
    _call("mmvae_layer_norm_bwd", _norm_args(
        x2, ldx, w, b, wtype, mean=mean.data_ptr(), rstd=rstd.data_ptr(), dy=dy2.data_ptr(), lddy=lddy,
        dx=dx.data_ptr() if need[0] else 0, lddx=N, dw=dw.data_ptr() if need[1] else 0, db=db.data_ptr() if need[2] else 0,
        ws=ws.data_ptr() if n else 0, ws_bytes=n, relu=relu, p=p, seed=seed, step=step, row_offset=row_offset, state=_state(state, x2)))
    return dx, dw, db


def dropout_apply(x, p, seed, *, step=0, row_offset=0, state=None):
    """x with each element dropped with probability p, or scaled by 1 / P(kept); on dy: the gradient."""
    x2, ldx = _rows(x, "x")
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    st, dev = _stream(x2)
    _call("mmvae_dropout", _DROP.pack(x2.shape[0], x2.shape[1], x2.data_ptr(), ldx, y.data_ptr(), x2.shape[1], p, seed & _MASK,
                                      step & _MASK, row_offset & _MASK, _state(state, x2), st, dev, _TYPE[x.dtype]))
    return y


def _ids(ids, device):
    if not isinstance(ids, torch.Tensor) or ids.dtype not in (torch.int64, torch.int32) or ids.device != device:
        _wrong("ids must be an int64 or int32 tensor on the table's device")
    return ids.contiguous()


def embedding_forward(ids, table, scale=1.0, add=None):
    """scale * table[ids] (+ add), ids of any shape; an id outside [0, rows) looks up zeros."""
    t2, ldt = _rows(table, "table")
    if table.dim() != 2:
        _wrong("table must be [rows, N]")
    i = _ids(ids, table.device)
    N = t2.shape[1]
    y = torch.empty((*ids.shape, N), dtype=table.dtype, device=table.device)
    a, lda = 0, 0
    if add is not None:
        a2, lda = _rows(add, "add", y)
        a = a2.data_ptr()
    st, dev = _stream(t2)
    _call("mmvae_embedding_fwd", _EMB.pack(i.numel(), N, t2.shape[0], i.data_ptr(), t2.data_ptr(), ldt, a, lda, y.data_ptr(), N, 0, 0, 0, 0,
                                           0, st, dev, _TYPE[table.dtype], 1 if i.dtype == torch.int64 else 0, scale))
    return y


def embedding_backward(dy, ids, rows, scale=1.0):
    """The table's gradient [rows, N] in dy's type: scale times the sum of dy over each row's tokens."""
    d2, lddy = _rows(dy, "dy")
    i = _ids(ids, dy.device)
    T, N = i.numel(), dy.shape[-1]
    if dy.shape[:-1] != ids.shape:
        _wrong("dy must be ids' shape and the width")
    if not isinstance(rows, int) or rows < 0:
        _wrong("rows must be the table's row count")
    out = torch.empty((rows, N), dtype=dy.dtype, device=dy.device)
    n = lib().mmvae_embedding_bwd_ws(T, N)
    ws = torch.empty(n, dtype=torch.uint8, device=dy.device)
    st, dev = _stream(d2)
    _call("mmvae_embedding_bwd", _EMB.pack(T, N, rows, i.data_ptr(), 0, 0, 0, 0, 0, 0, d2.data_ptr(), lddy, out.data_ptr(), ws.data_ptr(), n,
                                           st, dev, _TYPE[dy.dtype], 1 if i.dtype == torch.int64 else 0, scale))
    return out


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, kw):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps, stats=any(ctx.needs_input_grad[:3]), **kw)
        ctx.save_for_backward(x, weight, bias, mean, rstd, kw.get("state"))
        ctx.kw = kw
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, mean, rstd, _ = ctx.saved_tensors
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, weight, bias, need=ctx.needs_input_grad[:3], **ctx.kw)
        return dx, dw, db, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, relu=False, p=0.0, seed=0, step=0, row_offset=0, state=None):
    """drop(relu?(norm(x) * weight + bias)) over x's last dimension (differentiable in x, weight, bias).
    ``state`` must hold the forward's values when the backward runs."""
    return _LayerNorm.apply(x, weight, bias, eps, dict(relu=relu, p=p, seed=seed, step=step, row_offset=row_offset, state=state))


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, kw):
        ctx.key = (p, seed, kw)
        return dropout_apply(x, p, seed, **kw)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        p, seed, kw = ctx.key
        return dropout_apply(dy, p, seed, **kw), None, None, None


def dropout(x, p, seed, *, step=0, row_offset=0, state=None):
    """x with dropout (differentiable; the backward recomputes the mask from the same key)."""
    return _Dropout.apply(x, p, seed, dict(step=step, row_offset=row_offset, state=state))


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, add):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale = table.shape[0], scale
        return embedding_forward(ids, table, scale, add)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        dt = embedding_backward(dy, ids, ctx.rows, ctx.scale) if ctx.needs_input_grad[1] else None
        return None, dt, None, dy if ctx.needs_input_grad[3] else None


def embedding(ids, table, scale=1.0, add=None):
    """scale * table[ids] (+ add) (differentiable in table and add)."""
    return _Embedding.apply(ids, table, scale, add)
