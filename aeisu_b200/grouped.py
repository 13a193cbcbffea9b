"""Matrix products grouped by expert: rows sorted by expert, ragged group sizes, one launch.

The grouped layers of the controller give each channel group its own weights; here each *row* (a pixel
of a tile, a token) belongs to one of E experts.  ``offsets`` [E + 1] bounds the groups: rows
``offsets[e] : offsets[e + 1]`` of x are multiplied by ``weight[e]``.  The bounds stay on the GPU: the
call never waits for them, so it may be captured into a CUDA graph and replayed with other bounds
(a backward pass only while no eager graph of the same leaves lives, as for ``block_fp8``).

    y = grouped_matmul(x, weight, offsets)             # x [T, K], weight [E, N, K]: y [T, N]

Float weights (float16 or bfloat16, the type of x) train: gradients of x and weight are products of
the same kind, an expert without rows gets zeros.  BlockFP8 weights (``quantize(weight, rows=128)``)
serve: x is quantised in the call, or given as BlockFP8.  Sums are held in float32 and rounded once.
Rows in no group are zero, or, with ``out``, left as they were there.
``block_fp8.check_products()`` tells whether a kernel gave up a wait.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from . import _matrices as mx
from .block_fp8 import BlockFP8

MAX_GROUPS = 1024
_HALVES = (torch.float16, torch.bfloat16)
_call = _lib.lib
_pack = _lib.MATRIX.pack


def _weights(weight, flip=False):
    """(tensor kept, aeisu_matrix) of weights [E, N, K], or of their transposes [E, K, N], stored with either of
    the last two dimensions contiguous."""
    e, n, k = weight.shape
    at = weight.data_ptr()
    if weight.stride() == (n * k, k, 1) and k % 8 == 0 and at % 16 == 0 and (k > 1 or not flip):
        rows, cols = (k, n) if flip else (n, k)
        return weight, _pack(at, 0, mx.TYPES[weight.dtype], rows, cols, e, k, n * k, 0, flip)
    if flip:
        weight = weight.transpose(1, 2)
    other = weight.transpose(1, 2)
    if mx.row_stride(weight) is None and mx.row_stride(other) is not None:
        t, ld = mx.operand(other)
        return t, mx.matrix(t, ld, transposed=True)
    t, ld = mx.operand(weight)
    return t, mx.matrix(t, ld)


def _product(x, weight, offsets, out, ld, zero_outside):
    """x, weight: (tensors kept, aeisu_matrix); ld: elements from row to row of out."""
    index = out.get_device()
    _lib.check(_call().aeisu_grouped_product(x[1], weight[1], offsets.data_ptr(), zero_outside, mx.matrix(out, ld), index,
                                             mx.stream(index)))
    return out


def _rows(x):
    t, ld = mx.operand(x)
    return t, mx.matrix(t, ld)


class _Grouped(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets):
        t, n = x.shape[0], weight.shape[1]
        kept = _rows(x)      # an aligned copy serves the backward pass too
        ctx.save_for_backward(kept[0], weight, offsets)
        out = x.new_empty((t, n))
        return _product(kept, _weights(weight), offsets, out, n, True) if t else out

    @staticmethod
    def backward(ctx, grad):
        return _Grouped.twice(ctx, grad) if torch.is_grad_enabled() else _Grouped.once(ctx, grad)

    @staticmethod
    def once(ctx, grad):
        if forward_ad._current_level >= 0:
            mx.refuse_tangents("grouped_matmul", grad)
        x, weight, offsets = ctx.saved_tensors
        t, k = x.shape
        need_x, need_w, _ = ctx.needs_input_grad
        if t == 0:
            return x.new_empty((0, k)), torch.zeros_like(weight), None
        g = _rows(grad)
        gx = gw = None
        if need_x:
            gx = _product(g, _weights(weight, True), offsets, x.new_empty((t, k)), k, True)
        if need_w:
            gw = weight.new_empty(weight.shape)
            kept = _rows(x)
            index = gw.get_device()
            _lib.check(_call().aeisu_grouped_weight_gradient(g[1], kept[1], offsets.data_ptr(), weight.shape[0],
                                                             gw.data_ptr(), mx.TYPES[gw.dtype], index, mx.stream(index)))
        return gx, gw, None

    twice = staticmethod(once_differentiable(lambda ctx, grad: _Grouped.once(ctx, grad)))


def grouped_matmul(x, weight, offsets, *, out=None, dtype=None):
    """``x[t] @ weight[e].T`` for the group e of each row t; see the module's text.

    ``x`` [T, K]; ``weight`` [E, N, K], E at most 1024, either of its last two dimensions contiguous;
    ``offsets`` int32 [E + 1], not decreasing, within [0, T] (values outside are moved to the nearest
    allowed one).  The result has x's type; ``dtype`` names it where x is BlockFP8 (default bfloat16).
    ``out`` [T, N] takes the result instead of a new tensor; it must not overlap x, and no gradients flow
    through it.
    """
    fp8 = isinstance(weight, BlockFP8)
    coded = isinstance(x, BlockFP8)
    if coded and not fp8:
        raise TypeError("a BlockFP8 x needs BlockFP8 weights")
    if len(x.shape) != 2 or len(weight.shape) != 3 or x.shape[1] != weight.shape[2] or 0 in weight.shape:
        raise ValueError("Expected x [T, K] and weight [E, N, K]")
    (t, k), n = x.shape, weight.shape[1]
    if t > mx.MAX_SIDE or n > mx.MAX_SIDE or k > mx.MAX_SIDE:
        raise mx.too_large(max(t, n, k))
    if weight.shape[0] > MAX_GROUPS:
        raise ValueError(f"at most {MAX_GROUPS} experts; got {weight.shape[0]}")
    if not fp8 and (weight.dtype not in _HALVES or x.dtype != weight.dtype):
        raise TypeError(f"x and weight must both be float16 or bfloat16; got {x.dtype} and {weight.dtype}")
    if fp8 and not coded and x.dtype not in mx.FLOATS:
        raise TypeError(f"x must be float32, float16, bfloat16 or BlockFP8; got {x.dtype}")
    if dtype is not None and not coded:
        raise ValueError("dtype is for a BlockFP8 x: the result has x's type")
    if offsets.dtype != torch.int32 or tuple(offsets.shape) != (weight.shape[0] + 1,):
        raise ValueError(f"Expected offsets int32 [{weight.shape[0] + 1}]")
    dtype = (dtype or torch.bfloat16) if coded else x.dtype
    if dtype not in mx.FLOATS:
        raise TypeError(f"the result is float32, float16 or bfloat16; got {dtype}")
    if out is not None and (tuple(out.shape) != (t, n) or out.dtype != dtype or (t and mx.row_stride(out) is None) or
                            out.requires_grad):
        raise ValueError(f"Expected out [{t}, {n}] of {dtype} with contiguous rows and without gradient")
    if forward_ad._current_level >= 0:
        mx.refuse_tangents("grouped_matmul", None if coded else x, None if fp8 else weight, out)
    index = mx.need_cuda("grouped_matmul", x.codes if coded else x, weight.codes if fp8 else weight, offsets,
                         *(() if out is None else (out,)))
    if torch.is_grad_enabled() and ((not coded and x.requires_grad) or (not fp8 and weight.requires_grad)):
        if fp8 or out is not None:
            raise ValueError("FP8 weights and out serve without gradients")
        return _Grouped.apply(x, weight, offsets.contiguous())
    new = out is None
    if new:
        out = offsets.new_empty((t, n), dtype=dtype)
    if t == 0:
        return out
    ld = n if new else mx.row_stride(out)
    offsets = offsets.contiguous()
    if not fp8:
        return _product(_rows(x), _weights(weight), offsets, out, ld, new)
    if coded:
        return _product(x.matrix(), weight.matrix(), offsets, out, ld, new)
    stride = mx.row_stride(x)
    if stride is None:
        x = mx.plain(x.detach())
        stride = k
    size = _call().aeisu_grouped_linear_workspace(t, k)
    ws, (codes, mw) = mx.scratch(size, x), weight.matrix()
    _lib.check(_call().aeisu_grouped_linear(mx.matrix(x, stride), mw, offsets.data_ptr(), new, mx.matrix(out, ld),
                                            ws.data_ptr(), size, index, mx.stream(index)))
    return out


__all__ = ["grouped_matmul", "MAX_GROUPS"]
