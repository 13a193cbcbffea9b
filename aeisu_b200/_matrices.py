"""Tensors as the C ABI's ``aeisu_matrix``: layouts, alignment, workspaces and streams."""
from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from . import _lib

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 3, torch.float8_e5m2: 4}
FLOATS = (torch.float32, torch.float16, torch.bfloat16)
CODES = (torch.float8_e4m3fn, torch.float8_e5m2)
BLOCK = 128
MAX_SIDE = 2 ** 31 - 1025   # rows or columns, as in the library
_pack = _lib.MATRIX.pack


def too_large(side):
    """The error for a side above MAX_SIDE: rows and columns are counted in 32 bits."""
    return ValueError(f"matrix sizes are out of range: at most {MAX_SIDE} rows or columns; got {side}")


def blocks(n):
    return -(-n // BLOCK)


def stream(index):
    """Handle of the current stream of CUDA device `index`."""
    return torch._C._cuda_getCurrentRawStream(index)


def need_cuda(name, *tensors):
    """All tensors on one CUDA device; its index."""
    for t in tensors:
        if not t.is_cuda:
            raise ValueError(f"{name} needs CUDA tensors (there is no CPU path)")
    index = tensors[0].get_device()
    for t in tensors[1:]:
        if t.get_device() != index:
            raise ValueError(f"{name}: the tensors must be on one device")
    return index


def refuse_tangents(name, *tensors):
    """An input of forward-mode differentiation is refused: its tangent would be lost in silence.  (Called where
    forward_ad._current_level is 0 or more: unpack_dual alone would cost every call 0.7 us per tensor.)"""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{name} has no forward-mode derivatives")


def row_stride(t):
    """Elements from row to row of a tensor whose rows are contiguous and do not overlap, else None; None too for a
    view whose memory holds the negated values (the imaginary part of a conjugate)."""
    shape, strides = t.shape, t.stride()
    r, c = shape[-2], shape[-1]
    if (c > 1 and strides[-1] != 1) or t.is_neg():
        return None
    ld = strides[-2] if r > 1 else c
    if ld < c or (len(shape) == 3 and shape[0] > 1 and strides[0] < (r - 1) * ld + c):
        return None
    return ld


def plain(t):
    """t, or a contiguous copy that holds its values as they are."""
    return t.resolve_neg().contiguous()


def matrix(t, ld, scales=None, rows=0, transposed=False):
    """aeisu_matrix of a 2-D or 3-D tensor (of its last two dimensions' transpose when transposed)."""
    shape = t.shape
    batch, step = (shape[0], t.stride(0)) if len(shape) == 3 else (1, 0)
    r, c = shape[-2], shape[-1]
    if transposed:
        r, c = c, r
    return _pack(t.data_ptr(), 0 if scales is None else scales.data_ptr(), TYPES[t.dtype], r, c, batch, ld, step, rows,
                 transposed)


def operand(t):
    """(tensor, row stride) fit for a product: t itself where its rows are contiguous and start on 16-byte
    boundaries, else a copy."""
    ld = row_stride(t)
    size = t.dtype.itemsize
    if ld is not None and t.shape[-2] == 1:
        ld = -(-ld * size // 16) * 16 // size   # the stride of a single row is never taken
    if ld is None or ld * size % 16 or t.data_ptr() % 16 or (t.dim() == 3 and t.shape[0] > 1 and t.stride(0) * size % 16):
        per = 16 // size
        ld = -(-t.shape[-1] // per) * per
        copy = t.new_empty_strided(t.shape, (t.shape[-2] * ld, ld, 1)[-t.dim():])
        copy.copy_(t)
        t = copy
    return t, ld


@functools.lru_cache(maxsize=4096)
def product_bytes(m, n, k, index):
    return _lib.lib().aeisu_product_workspace(m, n, k, index)


@functools.lru_cache(maxsize=4096)
def linear_bytes(m, n, k, train, index):
    return _lib.lib().aeisu_linear_workspace(m, n, k, train, index)


@functools.lru_cache(maxsize=4096)
def kept_bytes(rows, cols, block_rows):
    return _lib.lib().aeisu_linear_kept_bytes(rows, cols, block_rows)


def scratch(size, like):
    return like.new_empty(size, dtype=torch.uint8)
