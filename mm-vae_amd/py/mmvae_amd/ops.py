"""Layer operators on torch tensors: layer norm (with ReLU and dropout in the same pass), dropout and
embedding lookup, forward and backward (the "layer operators" of include/mmvae_capi.h, called
through the C++ module _ops).

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

lib()  # (libmmvae.so first, from its place in the tree; _ops.so links it)
from . import _ops  # noqa: E402

_ops.set_error(MMVAEError)

# the C argument structs, member by member (8-byte members first: no padding), for calls of the C entries through
# lib(): lib().mmvae_dropout(DROPOUT_ARGS.pack(...)); the calls below go through _ops
NORM_ARGS = struct.Struct("=2q Q q 2Q Q q 2Q Q q Q q 2Q Q q d 3Q Q Q 3i f 2i")
DROPOUT_ARGS = struct.Struct("=2q Q q Q q d 3Q Q Q 2i")
EMBEDDING_ARGS = struct.Struct("=3q 2Q q Q q Q q Q q Q Q q Q 3i f")


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, *, relu=False, p=0.0, seed=0, step=0, row_offset=0, state=None, stats=True):
    """y, mean, rstd of drop(relu?(norm(x) * weight + bias)) over x's last dimension; ``stats=False`` (serving)
    stores no statistics and returns None for them."""
    return _ops.norm_forward(x, weight, bias, eps, relu, p, seed, step, row_offset, state, stats)


def layer_norm_backward(dy, x, mean, rstd, weight=None, bias=None, *, relu=False, p=0.0, seed=0, step=0, row_offset=0, state=None,
                        need=(True, True, True)):
    """dx, dweight, dbias (of weight's type, float32 without one; None where ``need`` says so) from the forward's
    x and statistics; ReLU and dropout as the forward had them (its bias is needed for the ReLU)."""
    return _ops.norm_backward(dy, x, mean, rstd, weight, bias, relu, p, seed, step, row_offset, state, need[0], need[1], need[2])


def dropout_apply(x, p, seed, *, step=0, row_offset=0, state=None):
    """x with each element dropped with probability p, or scaled by 1 / P(kept); on dy: the gradient."""
    return _ops.dropout(x, p, seed, step, row_offset, state)


def embedding_forward(ids, table, scale=1.0, add=None):
    """scale * table[ids] (+ add), ids of any shape; an id outside [0, rows) looks up zeros."""
    return _ops.embedding_forward(ids, table, scale, add)


def embedding_backward(dy, ids, rows, scale=1.0):
    """The table's gradient [rows, N] in dy's type: scale times the sum of dy over each row's tokens."""
    return _ops.embedding_backward(dy, ids, rows, scale)


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
        ctx.save_for_backward(kw.get("state"))  # (changed before the backward: refused)
        return dropout_apply(x, p, seed, **kw)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        p, seed, kw = ctx.key
        ctx.saved_tensors
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
