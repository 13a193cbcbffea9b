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
codes of input and weight are kept for the backward pass.  Gradients of gradients are not computed.

All tensors must be CUDA tensors on one device; work goes to that device's current stream and may be
captured into a CUDA graph.  float64 is refused rather than computed at a lower precision.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from . import _matrices as mx

_E8M0 = torch.float8_e8m0fnu


class BlockFP8:
    """FP8 codes ``[R, C]`` or ``[E, R, C]`` and their block scales.

    ``scales`` (``torch.float8_e8m0fnu``, contiguous) is ``[..., ceil(C / 128), ceil(R / rows)]``: the
    scales of one block column lie together.  ``rows`` is 1 or 128; the value of a code is
    ``codes[r, c] * scales[c // 128, r // rows]``.
    """
    __slots__ = ("codes", "scales", "rows")

    def __init__(self, codes, scales, rows=1):
        if rows not in (1, mx.BLOCK):
            raise ValueError("blocks have 1 or 128 rows")
        if codes.dtype not in mx.CODES:
            raise TypeError(f"codes must be float8_e4m3fn or float8_e5m2; got {codes.dtype}")
        if scales.dtype != _E8M0:
            raise TypeError(f"scales must be float8_e8m0fnu; got {scales.dtype}")
        if codes.dim() not in (2, 3):
            raise ValueError("Expected codes [R, C] or [E, R, C]")
        r, c = codes.shape[-2:]
        want = (*codes.shape[:-2], mx.blocks(c), -(-r // rows))
        if tuple(scales.shape) != want or not scales.is_contiguous():
            raise ValueError(f"Expected contiguous scales {list(want)}; got {list(scales.shape)}")
        if codes.device != scales.device:
            raise ValueError("codes and scales must be on one device")
        self.codes, self.scales, self.rows = codes, scales, rows

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
        """aeisu_matrix for a product; the tensors it points to have to be kept by the caller."""
        codes, ld = mx.operand(self.codes)
        return codes, mx.matrix(codes, ld, self.scales, self.rows)

    def __repr__(self):
        return f"BlockFP8({list(self.codes.shape)}, {self.codes.dtype}, rows={self.rows}, {self.codes.device})"


def _empty(shape, rows, dtype, device):
    codes = mx.empty_rows(shape, dtype, device)
    scales = torch.empty((*shape[:-2], mx.blocks(shape[-1]), -(-shape[-2] // rows)), dtype=torch.uint8, device=device)
    return BlockFP8(codes, scales.view(_E8M0), rows)


def _out(q):
    return mx.matrix(q.codes, -(-q.codes.shape[-1] // 16) * 16, q.scales, q.rows)


def _quantize(x, rows, dtype, both):
    if x.dim() not in (2, 3) or x.shape[-1] == 0:
        raise ValueError("Expected values [R, C] or [E, R, C]")
    if rows not in (1, mx.BLOCK):
        raise ValueError("blocks have 1 or 128 rows")
    if dtype not in mx.CODES:
        raise TypeError(f"codes must be float8_e4m3fn or float8_e5m2; got {dtype}")
    if x.dtype not in mx.FLOATS:
        raise TypeError(f"quantize takes float32, float16 or bfloat16; got {x.dtype}")
    mx.need_cuda("quantize", x)
    x = x.detach()
    ld = mx.row_stride(x)
    if ld is None:
        x = x.contiguous()
        ld = x.shape[-1]
    if both and x.shape[-2] == 0:
        raise ValueError("Expected values with at least one row")
    q = _empty(x.shape, rows, dtype, x.device)
    t = _empty((*x.shape[:-2], x.shape[-1], x.shape[-2]), rows, dtype, x.device) if both else None
    if x.numel():
        mt = None if t is None else _out(t)
        m, mq = mx.matrix(x, ld), _out(q)
        _lib.check(_lib.lib().aeisu_block_quantize(C.byref(m), rows, C.byref(mq), None if mt is None else C.byref(mt),
                                                   x.device.index, mx.stream(x.device)))
    return q, t


def quantize(x, *, rows=1, dtype=torch.float8_e4m3fn):
    """Values ``[R, C]`` or ``[E, R, C]`` (float32, float16 or bfloat16) as BlockFP8; no gradient."""
    return _quantize(x, rows, dtype, False)[0]


def quantize_both(x, *, rows=1, dtype=torch.float8_e4m3fn):
    """``(quantize(x), quantize(x.transpose(-1, -2)))`` from one read of x."""
    return _quantize(x, rows, dtype, True)


def _check_bias(bias, n):
    if bias is None:
        return
    if tuple(bias.shape) != (n,):
        raise ValueError(f"Expected bias [{n}]")
    if bias.dtype not in mx.FLOATS:
        raise TypeError(f"bias must be float32, float16 or bfloat16; got {bias.dtype}")


def matmul(a, b, *, bias=None, dtype=torch.bfloat16):
    """``a @ b.T + bias`` of BlockFP8 ``a`` [M, K] and ``b`` [N, K], rounded once to ``dtype``; no gradient."""
    if not isinstance(a, BlockFP8) or not isinstance(b, BlockFP8):
        raise TypeError("matmul takes BlockFP8 operands")
    if len(a.shape) != 2 or len(b.shape) != 2 or a.shape[1] != b.shape[1] or a.shape[1] == 0:
        raise ValueError("Expected operands [M, K] and [N, K]")
    if dtype not in mx.FLOATS:
        raise TypeError(f"matmul gives float32, float16 or bfloat16; got {dtype}")
    _check_bias(bias, b.shape[0])
    mx.need_cuda("matmul", a.codes, b.codes, *(() if bias is None else (bias,)))
    if a.shape[0] == 0 or b.shape[0] == 0:
        return torch.empty((a.shape[0], b.shape[0]), dtype=dtype, device=a.device)
    (ka, ma), (kb, mb) = a.matrix(), b.matrix()
    return mx.product(a.device, ma, mb, None if bias is None else bias.detach().contiguous(), dtype)


def _column_sum(x, dtype):
    lib = _lib.lib()
    out = torch.empty(x.shape[1], dtype=dtype, device=x.device)
    size = lib.aeisu_column_sum_workspace(*x.shape)
    ws = torch.empty(size, dtype=torch.uint8, device=x.device)
    m = mx.matrix(x, mx.row_stride(x))
    _lib.check(lib.aeisu_column_sum(C.byref(m), out.data_ptr(), mx.TYPES[dtype], ws.data_ptr(), size, x.device.index,
                                    mx.stream(x.device)))
    return out


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, grad_dtype):
        need_x, need_w = ctx.needs_input_grad[:2]
        ctx.sizes = x.shape, weight.shape
        ctx.types = (x.dtype, weight.dtype, None if bias is None else bias.dtype, grad_dtype)
        if x.shape[0] == 0:
            ctx.kept = None
            return x.new_empty(0, weight.shape[0])
        q, qt = _quantize(x, 1, torch.float8_e4m3fn, need_w)
        w, wt = _quantize(weight, mx.BLOCK, torch.float8_e4m3fn, need_x)
        ctx.kept = [None if t is None else t.rows for t in (qt, wt)]
        ctx.save_for_backward(*(None if t is None else v for t in (qt, wt) for v in (
            (None, None) if t is None else (t.codes, t.scales))))
        return matmul(q, w, bias=bias, dtype=x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x_type, w_type, b_type, grad_dtype = ctx.types
        if ctx.kept is None:   # no rows
            x_size, w_size = ctx.sizes
            return (grad.new_empty(x_size, dtype=x_type), grad.new_zeros(w_size, dtype=w_type),
                    None if b_type is None else grad.new_zeros(w_size[0], dtype=b_type), None)
        saved = ctx.saved_tensors
        qt, wt = (None if rows is None else BlockFP8(saved[2 * i], saved[2 * i + 1], rows)
                  for i, rows in enumerate(ctx.kept))
        if mx.row_stride(grad) is None:
            grad = grad.contiguous()
        gx = gw = gb = None
        if qt is not None:
            g, gt = _quantize(grad, 1, grad_dtype, True)
            gw = matmul(gt, qt, dtype=w_type)
        elif wt is not None:
            g = quantize(grad, dtype=grad_dtype)
        if wt is not None:
            gx = matmul(g, wt, dtype=x_type)
        if ctx.needs_input_grad[2]:
            gb = _column_sum(grad, b_type)
        return gx, gw, gb, None


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
    if x.dim() < 1 or len(weight.shape) != 2 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError("Expected x [..., K] and weight [N, K]")
    _check_bias(bias, weight.shape[0])
    mx.need_cuda("linear", x, weight.codes if serving else weight, *(() if bias is None else (bias,)))
    wants = torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                            for t in (x, None if serving else weight, bias))
    if serving and wants:
        raise ValueError("FP8 weights serve without gradients: pass the float weight to train")
    lead = x.shape[:-1]
    flat = x.reshape(lead.numel(), x.shape[-1])
    with torch.autocast(device_type="cuda", enabled=False):
        if wants:
            y = _Linear.apply(flat, weight, bias, grad_dtype)
        else:
            w = weight if serving else quantize(weight, rows=mx.BLOCK)
            y = matmul(quantize(flat), w, bias=bias, dtype=x.dtype)
    return y.reshape(*lead, weight.shape[0])


__all__ = ["BlockFP8", "quantize", "quantize_both", "matmul", "linear"]
