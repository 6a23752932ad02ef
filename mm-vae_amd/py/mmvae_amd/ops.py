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


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _rows(t, name):
    """t as [rows, N] with unit column stride (a view where it is one)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _wrong(f"{name} must be a CUDA tensor")
    if t.dtype not in _TYPE:
        _wrong(f"{name}: float32, bfloat16 or float16, not {t.dtype}")
    if t.dim() == 0 or t.shape[-1] == 0:
        _wrong(f"{name} needs a last dimension of at least 1")
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1 and t.shape[1] > 1:
        t = t.contiguous()
    return t


def _like(t, name, x):
    if not isinstance(t, torch.Tensor) or t.shape != x.shape or t.dtype != x.dtype or t.get_device() != x.get_device():
        _wrong(f"{name} must have the shape, type and device of the other tensors")


def _weight(t, name, N, x):
    """Pointer and type code of a weight or bias."""
    if not isinstance(t, torch.Tensor) or t.get_device() != x.get_device() or t.dim() != 1 or t.shape[0] != N:
        _wrong(f"{name} must be a tensor of [{N}] on x's device")
    if t.dtype != x.dtype and t.dtype != torch.float32:
        _wrong(f"{name}: x's type or float32, not {t.dtype}")
    if not t.is_contiguous():
        _wrong(f"{name} must be contiguous")
    return t.data_ptr(), _TYPE[t.dtype]


def _weights(weight, bias, N, x):
    """(weight pointer, bias pointer, their type code)"""
    w = b = 0
    tw = tb = -1
    if weight is not None:
        w, tw = _weight(weight, "weight", N, x)
    if bias is not None:
        b, tb = _weight(bias, "bias", N, x)
        if tw >= 0 and tw != tb:
            _wrong("weight and bias must have one type")
    return w, b, max(tw, tb, 0)


def _state(state, x):
    if (not isinstance(state, torch.Tensor) or state.get_device() != x.get_device() or state.dtype != torch.int64 or state.numel() != 2
            or not state.is_contiguous()):
        _wrong("state must be a contiguous int64 tensor [step, row_offset] on x's device")
    return state.data_ptr()


def _failed(name, rc):
    _wrong(f"{name} failed ({rc}): {lib().mmvae_last_error(None).decode()}")


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, *, relu=False, p=0.0, seed=0, step=0, row_offset=0, state=None, stats=True):
    """y, mean, rstd of drop(relu?(norm(x) * weight + bias)) over x's last dimension; ``stats=False`` (serving)
    stores no statistics and returns None for them."""
    x2 = _rows(x, "x")
    M, N = x2.shape
    w, b, wtype = _weights(weight, bias, N, x2)
    y = x.new_empty(x.shape)
    mean = rstd = None
    pm = pr = 0
    if stats:
        mean, rstd = x.new_empty(x.shape[:-1], dtype=torch.float32), x.new_empty(x.shape[:-1], dtype=torch.float32)
        pm, pr = mean.data_ptr(), rstd.data_ptr()
    dev = x2.get_device()
    rc = lib().mmvae_layer_norm_fwd(_NORM.pack(
        M, N, x2.data_ptr(), x2.stride(0), w, b, y.data_ptr(), N, pm, pr, 0, 0, 0, 0, 0, 0, 0, 0, p, seed & _MASK, step & _MASK,
        row_offset & _MASK, 0 if state is None else _state(state, x2), _raw_stream(dev), dev, _TYPE[x2.dtype], wtype, eps, 1 if relu else 0, 0))
    if rc:
        _failed("layer_norm_forward", rc)
    return y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight=None, bias=None, *, relu=False, p=0.0, seed=0, step=0, row_offset=0, state=None,
                        need=(True, True, True)):
    """dx, dweight, dbias (of weight's type, float32 without one; None where ``need`` says so) from the forward's
    x and statistics; ReLU and dropout as the forward had them (its bias is needed for the ReLU)."""
    x2 = _rows(x, "x")
    _like(dy, "dy", x)
    dy2 = _rows(dy, "dy")
    M, N = x2.shape
    w, b, wtype = _weights(weight, bias, N, x2)
    dev = x2.get_device()
    for t in (mean, rstd):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.get_device() != dev or t.numel() != M or not t.is_contiguous():
            _wrong("mean and rstd must be the forward's float32 statistics")
    wt = weight if weight is not None else bias
    wt = torch.float32 if wt is None else wt.dtype
    dx = x.new_empty(x.shape) if need[0] else None
    dw = x.new_empty((N,), dtype=wt) if need[1] else None
    db = x.new_empty((N,), dtype=wt) if need[2] else None
    ws, n = None, 0
    if need[1] or need[2]:
        n = lib().mmvae_layer_norm_bwd_ws(M, N)
        if n:
            ws = x.new_empty((n,), dtype=torch.uint8)
    rc = lib().mmvae_layer_norm_bwd(_NORM.pack(
        M, N, x2.data_ptr(), x2.stride(0), w, b, 0, 0, mean.data_ptr(), rstd.data_ptr(), dy2.data_ptr(), dy2.stride(0),
        dx.data_ptr() if need[0] else 0, N, dw.data_ptr() if need[1] else 0, db.data_ptr() if need[2] else 0, ws.data_ptr() if n else 0, n,
        p, seed & _MASK, step & _MASK, row_offset & _MASK, 0 if state is None else _state(state, x2), _raw_stream(dev), dev, _TYPE[x2.dtype],
        wtype, 0.0, 1 if relu else 0, 0))
    if rc:
        _failed("layer_norm_backward", rc)
    return dx, dw, db


def dropout_apply(x, p, seed, *, step=0, row_offset=0, state=None):
    """x with each element dropped with probability p, or scaled by 1 / P(kept); on dy: the gradient."""
    x2 = _rows(x, "x")
    y = x.new_empty(x.shape)
    M, N = x2.shape
    dev = x2.get_device()
    rc = lib().mmvae_dropout(_DROP.pack(M, N, x2.data_ptr(), x2.stride(0), y.data_ptr(), N, p, seed & _MASK, step & _MASK, row_offset & _MASK,
                                        0 if state is None else _state(state, x2), _raw_stream(dev), dev, _TYPE[x2.dtype]))
    if rc:
        _failed("dropout_apply", rc)
    return y


def _ids(ids, t):
    if not isinstance(ids, torch.Tensor) or ids.dtype not in (torch.int64, torch.int32) or ids.get_device() != t.get_device():
        _wrong("ids must be an int64 or int32 tensor on the table's device")
    return ids if ids.is_contiguous() else ids.contiguous()


def embedding_forward(ids, table, scale=1.0, add=None):
    """scale * table[ids] (+ add), ids of any shape; an id outside [0, rows) looks up zeros."""
    t2 = _rows(table, "table")
    if table.dim() != 2:
        _wrong("table must be [rows, N]")
    i = _ids(ids, t2)
    V, N = t2.shape
    y = t2.new_empty((*ids.shape, N))
    a = lda = 0
    if add is not None:
        _like(add, "add", y)
        add = _rows(add, "add")
        a, lda = add.data_ptr(), add.stride(0)
    dev = t2.get_device()
    rc = lib().mmvae_embedding_fwd(_EMB.pack(i.numel(), N, V, i.data_ptr(), t2.data_ptr(), t2.stride(0), a, lda, y.data_ptr(), N, 0, 0, 0, 0, 0,
                                             _raw_stream(dev), dev, _TYPE[t2.dtype], 1 if i.dtype == torch.int64 else 0, scale))
    if rc:
        _failed("embedding_forward", rc)
    return y


def embedding_backward(dy, ids, rows, scale=1.0):
    """The table's gradient [rows, N] in dy's type: scale times the sum of dy over each row's tokens."""
    d2 = _rows(dy, "dy")
    i = _ids(ids, d2)
    T, N = i.numel(), dy.shape[-1]
    if dy.shape[:-1] != ids.shape:
        _wrong("dy must be ids' shape and the width")
    if not isinstance(rows, int) or rows < 0:
        _wrong("rows must be the table's row count")
    out = d2.new_empty((rows, N))
    n = lib().mmvae_embedding_bwd_ws(T, N, rows)
    ws = d2.new_empty((n,), dtype=torch.uint8)
    dev = d2.get_device()
    rc = lib().mmvae_embedding_bwd(_EMB.pack(T, N, rows, i.data_ptr(), 0, 0, 0, 0, 0, 0, d2.data_ptr(), d2.stride(0), out.data_ptr(), ws.data_ptr(), n,
                                             _raw_stream(dev), dev, _TYPE[d2.dtype], 1 if i.dtype == torch.int64 else 0, scale))
    if rc:
        _failed("embedding_backward", rc)
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
