"""Block-scaled FP8: quantisation, products and a trainable linear layer on tcgen05.

The SPYR8 artifact gives an FP8 layer one scale per activation tensor and one per output channel.
For wide layers and for training that is too coarse: here every block of 128 values of a row (of
``128 x 128`` values of a weight) has a scale of its own.  Scales are powers of two (E8M0), so that
scaling is exact and the tensor core applies them inside the product.

    q = quantize(x)                        # BlockFP8: codes [R, C], one scale per 1 x 128 values
    w = quantize(weight, rows=128)         # one scale per 128 x 128 values
    y = matmul(q, w, bias=bias)            # x @ weight.T + bias
    y = linear(x, weight, bias)            # the same from float tensors, with gradients
    y = linear(x, w, bias)                 # serving: the weights stay in FP8

Arithmetic: the scale of a block is the smallest power of two ``s`` with ``amax / s`` no larger than
the largest finite code (448 for E4M3, 57344 for E5M2), 1 for a block of zeros; a code is ``x / s``
rounded to nearest even.  Infinities and NaN become NaN codes and do not count for ``amax``.  Products
accumulate in float32 and round once to the output's type; repeated calls give the same bits.

``linear`` trains: the input gradient is the product of the gradient's rows with the weight's blocks,
the weight gradient that of the gradient's columns with the input's columns (blocks of 128 rows of
the batch), both operands in FP8; the bias gradient is summed in float32.  Only the transposed FP8
codes of input and weight are kept for the backward pass.  Gradients of gradients and forward-mode
derivatives are not computed: both are refused.

All tensors must be CUDA tensors on one device; work goes to that device's current stream and may be
captured into a CUDA graph.  A backward pass is captured only while no eager graph of the same leaves
lives: torch would make the capture wait for that graph's stream, and the capture fails.  float64 is
refused rather than computed at a lower precision.

The waits inside the product kernel are bounded: one that makes no progress for about two seconds ends
its kernel, whose outputs are then undefined.  ``check_products()`` waits for the device and raises if that
has happened; call it where a program synchronises anyway.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from . import _matrices as mx

_E8M0 = torch.float8_e8m0fnu
_call = _lib.lib
_new = object.__new__
_pack = _lib.MATRIX.pack
_MOST = mx.MAX_SIDE


@functools.lru_cache(maxsize=4096)
def _sizes(shape, rows):
    """(row stride of the codes, shape of the codes' storage, shape of the scales)."""
    *lead, r, c = shape
    if max(r, c) > _MOST:
        raise mx.too_large(max(r, c))
    ld = -(-c // 16) * 16
    return ld, (*lead, r, ld), (*lead, mx.blocks(c), -(-r // rows))


def _form(codes, ld, rows):
    """The fields of aeisu_matrix behind its pointers; None where a product has to take a copy."""
    shape = codes.shape
    batch, step = (shape[0], codes.stride(0)) if len(shape) == 3 else (1, 0)
    r, c = shape[-2], shape[-1]
    if ld is not None and r == 1:
        ld = -(-ld // 16) * 16   # the stride of a single row is never taken
    if ld is None or ld % 16 or (batch > 1 and step % 16):
        return None
    return mx.TYPES[codes.dtype], r, c, batch, ld, step, rows, 0


def _empty(x, shape, rows, dtype):
    """(uninitialised BlockFP8 beside x, its aeisu_matrix)."""
    ld, stored, scaled = _sizes(shape, rows)
    q = _new(BlockFP8)
    codes = x.new_empty(stored, dtype=dtype)
    at = codes.data_ptr()
    q._codes = codes = codes if ld == shape[-1] else codes[..., :shape[-1]]
    q._scales = scales = x.new_empty(scaled, dtype=_E8M0)
    q._rows = rows
    q._form = form = _form(codes, ld, rows)
    return q, _pack(at, scales.data_ptr(), *form)


class BlockFP8:
    """FP8 codes ``[R, C]`` or ``[E, R, C]`` and their block scales.

    ``scales`` (``torch.float8_e8m0fnu``, contiguous) is ``[..., ceil(C / 128), ceil(R / rows)]``: the
    scales of one block column lie together.  ``rows`` is 1 or 128; the value of a code is
    ``codes[r, c] * scales[c // 128, r // rows]``.  The tensors' values may change, their sizes and strides
    may not.
    """
    __slots__ = ("_codes", "_scales", "_rows", "_form")

    def __init__(self, codes, scales, rows=1):
        if rows != 1 and rows != mx.BLOCK:
            raise ValueError("blocks have 1 or 128 rows")
        if codes.dtype not in mx.CODES:
            raise TypeError(f"codes must be float8_e4m3fn or float8_e5m2; got {codes.dtype}")
        if scales.dtype != _E8M0:
            raise TypeError(f"scales must be float8_e8m0fnu; got {scales.dtype}")
        shape = codes.shape
        if len(shape) != 2 and len(shape) != 3:
            raise ValueError("Expected codes [R, C] or [E, R, C]")
        want = _sizes(shape, rows)[2]
        if scales.shape != want or not scales.is_contiguous():
            raise ValueError(f"Expected contiguous scales {list(want)}; got {list(scales.shape)}")
        if codes.get_device() != scales.get_device():
            raise ValueError("codes and scales must be on one device")
        self._codes, self._scales, self._rows = codes, scales, rows
        self._form = _form(codes, mx.row_stride(codes), rows)

    @property
    def codes(self):
        return self._codes

    @property
    def scales(self):
        return self._scales

    @property
    def rows(self):
        return self._rows

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    def dequantize(self):
        """The values as float32."""
        r, c = self.codes.shape[-2:]
        s = self.scales.to(torch.float32).transpose(-1, -2)
        s = s.repeat_interleave(self.rows, -2)[..., :r, :].repeat_interleave(mx.BLOCK, -1)[..., :c]
        return self.codes.to(torch.float32) * s

    def matrix(self):
        """(codes, aeisu_matrix) for a product; the codes, a copy where theirs do not start rows on 16-byte
        boundaries, have to be kept by the caller."""
        codes, form = self._codes, self._form
        at = codes.data_ptr()
        if form is None or at % 16:
            codes, ld = mx.operand(codes)
            return codes, mx.matrix(codes, ld, self._scales, self._rows)
        return codes, _pack(at, self._scales.data_ptr(), *form)

    def __repr__(self):
        return f"BlockFP8({list(self.codes.shape)}, {self.codes.dtype}, rows={self.rows}, {self.codes.device})"


def _quantize(x, rows, dtype, both):
    shape = x.shape
    if len(shape) not in (2, 3) or shape[-1] == 0:
        raise ValueError("Expected values [R, C] or [E, R, C]")
    if rows not in (1, mx.BLOCK):
        raise ValueError("blocks have 1 or 128 rows")
    if shape[-2] > _MOST or shape[-1] > _MOST:
        raise mx.too_large(max(shape[-2:]))
    if dtype not in mx.CODES:
        raise TypeError(f"codes must be float8_e4m3fn or float8_e5m2; got {dtype}")
    if x.dtype not in mx.FLOATS:
        raise TypeError(f"quantize takes float32, float16 or bfloat16; got {x.dtype}")
    index = mx.need_cuda("quantize", x)
    ld = mx.row_stride(x)
    if ld is None:
        x = mx.plain(x.detach())
        ld = shape[-1]
    q, mq = _empty(x, tuple(shape), rows, dtype)
    t = mt = None
    if both:
        if shape[-2] == 0:
            raise ValueError("Expected values with at least one row")
        t, mt = _empty(x, (*shape[:-2], shape[-1], shape[-2]), rows, dtype)
    if x.numel():
        _lib.check(_call().aeisu_block_quantize(mx.matrix(x, ld), rows, mq, mt, index, mx.stream(index)))
    return q, t


def quantize(x, *, rows=1, dtype=torch.float8_e4m3fn):
    """Values ``[R, C]`` or ``[E, R, C]`` (float32, float16 or bfloat16) as BlockFP8; no gradient."""
    return _quantize(x, rows, dtype, False)[0]


def quantize_both(x, *, rows=1, dtype=torch.float8_e4m3fn):
    """``(quantize(x), quantize(x.transpose(-1, -2)))`` from one read of x."""
    return _quantize(x, rows, dtype, True)


def _bias(bias, n):
    """The bias ready for the library; None without one."""
    if bias is None:
        return None
    if tuple(bias.shape) != (n,):
        raise ValueError(f"Expected bias [{n}]")
    if bias.dtype not in mx.FLOATS:
        raise TypeError(f"bias must be float32, float16 or bfloat16; got {bias.dtype}")
    return bias if (n == 1 or bias.stride(0) == 1) and not bias.is_neg() else mx.plain(bias)


def matmul(a, b, *, bias=None, dtype=torch.bfloat16):
    """``a @ b.T + bias`` of BlockFP8 ``a`` [M, K] and ``b`` [N, K], rounded once to ``dtype``; no gradient."""
    if not isinstance(a, BlockFP8) or not isinstance(b, BlockFP8):
        raise TypeError("matmul takes BlockFP8 operands")
    if len(a.shape) != 2 or len(b.shape) != 2 or a.shape[1] != b.shape[1] or a.shape[1] == 0:
        raise ValueError("Expected operands [M, K] and [N, K]")
    if dtype not in mx.FLOATS:
        raise TypeError(f"matmul gives float32, float16 or bfloat16; got {dtype}")
    (m, k), n = a.shape, b.shape[0]
    bias = _bias(bias, n)
    index = mx.need_cuda("matmul", a.codes, b.codes, *(() if bias is None else (bias,)))
    out = a.codes.new_empty((m, n), dtype=dtype)
    if m == 0 or n == 0:
        return out
    (ka, ma), (kb, mb) = a.matrix(), b.matrix()
    size = mx.product_bytes(m, n, k, index)
    ws = mx.scratch(size, out) if size else None
    _lib.check(_call().aeisu_product(ma, mb, None if bias is None else bias.data_ptr(),
                                        0 if bias is None else mx.TYPES[bias.dtype], mx.matrix(out, n),
                                        None if ws is None else ws.data_ptr(), size, index, mx.stream(index)))
    return out


def _rows(x):
    """(tensor, aeisu_matrix) of values whose rows may start anywhere."""
    ld = mx.row_stride(x)
    if ld is None:
        x = mx.plain(x)
        ld = x.shape[-1]
    return x, mx.matrix(x, ld)


def _forward(x, weight, bias, kept_x, kept_w, index):
    """The layer on float x and weight, leaving the transposed codes at the addresses kept_x and kept_w."""
    (m, k), n = x.shape, weight.shape[0]
    out = x.new_empty((m, n))
    size = mx.linear_bytes(m, n, k, 1, index)
    ws = mx.scratch(size, out)
    (x, mat), (weight, mw) = _rows(x), _rows(weight)
    _lib.check(_call().aeisu_linear_forward(
        mat, mw, None if bias is None else bias.data_ptr(), 0 if bias is None else mx.TYPES[bias.dtype],
        mx.matrix(out, n), kept_x, kept_w, ws.data_ptr(), size, index, mx.stream(index)))
    return out


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, grad_dtype):
        (m, k), n = x.shape, weight.shape[0]
        ctx.sizes = m, n, k
        ctx.types = (x.dtype, weight.dtype, None if bias is None else bias.dtype, grad_dtype)
        need_x, need_w = ctx.needs_input_grad[:2]
        if m == 0:
            return x.new_empty(0, n)
        size_x = mx.kept_bytes(m, k, 1) if need_w else 0
        size_w = mx.kept_bytes(n, k, mx.BLOCK) if need_x else 0
        kept = mx.scratch(size_x + size_w, x)
        ctx.save_for_backward(kept)
        ctx.places = (0 if need_w else None, size_x if need_x else None)
        at = kept.data_ptr()
        return _forward(x, weight, bias, at if need_w else None, at + size_x if need_x else None, x.get_device())

    @staticmethod
    def backward(ctx, grad):
        return _Linear.twice(ctx, grad) if torch.is_grad_enabled() else _Linear.once(ctx, grad)

    @staticmethod
    def once(ctx, grad):
        if forward_ad._current_level >= 0:
            mx.refuse_tangents("linear", grad)
        x_type, w_type, b_type, grad_dtype = ctx.types
        (m, n, k), (need_x, need_w, need_b, _), index = ctx.sizes, ctx.needs_input_grad, grad.get_device()
        new = grad.new_zeros if m == 0 else grad.new_empty
        gx = new((m, k), dtype=x_type) if need_x else None
        gw = new((n, k), dtype=w_type) if need_w else None
        gb = new((n,), dtype=b_type) if need_b else None
        if m == 0:
            return gx, gw, gb, None
        (kept,) = ctx.saved_tensors
        at = kept.data_ptr()
        kept_x, kept_w = ctx.places
        kept_x = None if kept_x is None else at + kept_x
        kept_w = None if kept_w is None else at + kept_w
        grad, mg = _rows(grad)
        size = mx.linear_bytes(m, n, k, 2, index)
        ws = mx.scratch(size, grad)
        _lib.check(_call().aeisu_linear_backward(
            mg, k, mx.TYPES[grad_dtype], kept_x, kept_w, gx.data_ptr() if need_x else None, mx.TYPES[x_type],
            gw.data_ptr() if need_w else None, mx.TYPES[w_type], gb.data_ptr() if need_b else None,
            mx.TYPES[b_type] if need_b else 0,
            ws.data_ptr(), size, index, mx.stream(index)))
        return gx, gw, gb, None

    twice = staticmethod(once_differentiable(lambda ctx, grad: _Linear.once(ctx, grad)))


def linear(x, weight, bias=None, *, grad_dtype=torch.float8_e4m3fn):
    """``x @ weight.T + bias`` with both operands in block-scaled FP8 (E4M3); ``x`` [..., K].

    ``weight`` is a float tensor [N, K], quantised in 128 x 128 blocks in the call and given a gradient,
    or a BlockFP8 kept from before, which serves without gradients.  The output has x's type; gradients
    have the types of their tensors.  ``grad_dtype`` is the FP8 type that the upstream gradient takes.
    """
    serving = isinstance(weight, BlockFP8)
    if x.dtype not in mx.FLOATS:
        raise TypeError(f"linear takes float32, float16 or bfloat16; got {x.dtype}")
    if not serving and weight.dtype not in mx.FLOATS:
        raise TypeError(f"weight must be float32, float16, bfloat16 or BlockFP8; got {weight.dtype}")
    if grad_dtype not in mx.CODES:
        raise TypeError(f"grad_dtype must be float8_e4m3fn or float8_e5m2; got {grad_dtype}")
    values = weight.codes if serving else weight
    shape, wide = x.shape, values.shape
    if len(shape) < 1 or len(wide) != 2 or shape[-1] != wide[1] or 0 in wide:
        raise ValueError("Expected x [..., K] and weight [N, K]")
    if forward_ad._current_level >= 0:
        mx.refuse_tangents("linear", x, None if serving else weight, bias)
    n, k = wide
    m = shape[0] if len(shape) == 2 else shape[:-1].numel()
    if m > _MOST or n > _MOST or k > _MOST:
        raise mx.too_large(max(m, n, k))
    if bias is None:
        ready = None
        index = mx.need_cuda("linear", x, values)
    else:
        ready = _bias(bias, n)
        index = mx.need_cuda("linear", x, values, bias)
    flat = x if len(shape) == 2 else x.reshape(m, k)
    if torch.is_grad_enabled() and (x.requires_grad or (not serving and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        if serving:
            raise ValueError("FP8 weights serve without gradients: pass the float weight to train")
        y = _Linear.apply(flat, weight, ready, grad_dtype)
    elif m == 0:
        y = flat.new_empty(0, n)
    elif not serving:
        y = _forward(flat, weight, ready, None, None, index)
    else:
        y = flat.new_empty((m, n))
        size = mx.linear_bytes(m, n, k, 0, index)
        ws = mx.scratch(size, flat)
        (flat, mat), (codes, mw) = _rows(flat), weight.matrix()
        _lib.check(_call().aeisu_linear(mat, mw, None if ready is None else ready.data_ptr(),
                                           0 if ready is None else mx.TYPES[ready.dtype], mx.matrix(y, n), ws.data_ptr(),
                                           size, index, mx.stream(index)))
    return y if len(shape) == 2 else y.reshape(*shape[:-1], n)


def check_products(device=None):
    """Waits for a CUDA device (default: the current one); ``TimeoutError`` if a product kernel on it, of this module or
    of ``grouped``, gave up a wait since the last call, so that outputs since then are undefined."""
    if device is None or isinstance(device, int):
        index = device
    else:
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"check_products needs a CUDA device; got {device}")
        index = device.index
    if index is None:
        index = torch.cuda.current_device()
    code = ctypes.c_int(0)
    _lib.check(_call().aeisu_product_status(index, ctypes.byref(code)))
    if code.value:
        raise TimeoutError(f"a product kernel on CUDA device {index} gave up a wait; outputs since the last check are undefined")


__all__ = ["BlockFP8", "quantize", "quantize_both", "matmul", "linear", "check_products"]
