"""Tensors as the C ABI's ``aeisu_matrix``: layouts, alignment and the calls shared by the products."""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 3, torch.float8_e5m2: 4}
FLOATS = (torch.float32, torch.float16, torch.bfloat16)
CODES = (torch.float8_e4m3fn, torch.float8_e5m2)
BLOCK = 128


def blocks(n):
    return -(-n // BLOCK)


def stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def need_cuda(name, *tensors):
    """All tensors on one CUDA device."""
    for t in tensors:
        if not t.is_cuda:
            raise ValueError(f"{name} needs CUDA tensors (there is no CPU path)")
        if t.device != tensors[0].device:
            raise ValueError(f"{name}: the tensors must be on one device")


def row_stride(t):
    """Elements from row to row of a tensor whose rows are contiguous and do not overlap, else None."""
    r, c = t.shape[-2:]
    if c > 1 and t.stride(-1) != 1:
        return None
    ld = t.stride(-2) if r > 1 else c
    if ld < c or (t.dim() == 3 and t.shape[0] > 1 and t.stride(0) < (r - 1) * ld + c):
        return None
    return ld


def matrix(t, ld, scales=None, rows=0, transposed=False):
    """aeisu_matrix of a 2-D or 3-D tensor (of its last two dimensions' transpose when transposed)."""
    batch = t.shape[0] if t.dim() == 3 else 1
    r, c = t.shape[-2:]
    if transposed:
        r, c = c, r
    return _lib.Matrix(t.data_ptr(), None if scales is None else scales.data_ptr(), TYPES[t.dtype], r, c, batch, ld,
                       t.stride(0) if batch > 1 else 0, rows, int(transposed))


def empty_rows(shape, dtype, device):
    """An uninitialised tensor whose rows start on 16-byte boundaries."""
    per = 16 // torch.empty((), dtype=dtype).element_size()
    c = shape[-1]
    return torch.empty((*shape[:-1], -(-c // per) * per), dtype=dtype, device=device)[..., :c]


def operand(t):
    """(tensor, row stride) fit for a product: t itself where its rows are contiguous and start on 16-byte
    boundaries, else a copy."""
    ld = row_stride(t)
    size = t.element_size()
    if ld is not None and t.shape[-2] == 1:
        ld = -(-ld * size // 16) * 16 // size   # the stride of a single row is never taken
    if ld is None or ld * size % 16 or t.data_ptr() % 16 or (t.dim() == 3 and t.shape[0] > 1 and t.stride(0) * size % 16):
        copy = empty_rows(t.shape, t.dtype, t.device)
        copy.copy_(t)
        t = copy
        ld = t.stride(-2)
    return t, ld


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(m, n, k, fp8, device):
    return _lib.lib().aeisu_product_workspace(m, n, k, fp8, device)


def product(device, ma, mb, bias, dtype):
    """a @ b.T (+ bias) of two aeisu_matrix operands on the device's current stream."""
    out = torch.empty((ma.rows, mb.rows), dtype=dtype, device=device)
    size = _workspace_bytes(ma.rows, mb.rows, ma.cols, int(ma.type >= 3), device.index)
    ws = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    mo = matrix(out, mb.rows)
    _lib.check(_lib.lib().aeisu_product(
        C.byref(ma), C.byref(mb), None if bias is None else bias.data_ptr(),
        0 if bias is None else TYPES[bias.dtype], C.byref(mo), None if ws is None else ws.data_ptr(), size,
        device.index, stream(device)))
    return out
