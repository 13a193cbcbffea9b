"""Block-scaled FP8 and grouped products without a GPU: the format, the refusals of the Python entry
points and those of the C entry points that come before any CUDA call."""
import ctypes as C

import pytest
import torch

import block_oracle as O
from aeisu_b200 import _lib, build
from aeisu_b200 import _matrices as mx
from aeisu_b200 import block_fp8 as B
from aeisu_b200.grouped import MAX_GROUPS, grouped_matmul

E4, E5, E8 = torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def scales(*shape):
    return torch.full(shape, 127, dtype=torch.uint8).view(E8)


def blocks(r, c, rows=1, dtype=E4, lead=()):
    return B.BlockFP8(torch.zeros(*lead, r, c).to(dtype), scales(*lead, -(-c // 128), -(-r // rows)), rows)


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dtype", [E4, E5])
def test_dequantize_is_codes_times_scales(rows, dtype):
    x = torch.randn(200, 300, generator=torch.Generator().manual_seed(1))
    v, s = O.quantize(x, rows, dtype)
    e = (torch.log2(s) + 127).to(torch.uint8).t().contiguous().view(E8)
    q = B.BlockFP8(v.to(dtype), e, rows)
    assert torch.equal(q.dequantize().double(), O.values(x, rows, dtype))
    # a code is off by at most half a step of its type, relative to the value, or of the least normal code
    half = torch.finfo(dtype).eps / 2
    least = s.repeat_interleave(rows, 0)[:200].repeat_interleave(128, 1)[:, :300] * 2.0 ** O.TOP[dtype][2]
    assert bool(((q.dequantize().double() - x.double()).abs() <= half * torch.maximum(x.double().abs(), least)).all())


def test_block_fp8_refuses_what_is_no_operand():
    codes = torch.zeros(10, 300).to(E4)
    B.BlockFP8(codes, scales(3, 10))
    for bad in (scales(3, 9), scales(10, 3), scales(2, 10), scales(3, 20)[:, ::2], scales(1, 3, 10)):
        with pytest.raises(ValueError, match="scales"):
            B.BlockFP8(codes, bad)
    with pytest.raises(ValueError, match="1 or 128"):
        B.BlockFP8(codes, scales(3, 1), 64)
    with pytest.raises(TypeError, match="codes"):
        B.BlockFP8(torch.zeros(10, 300), scales(3, 10))
    with pytest.raises(TypeError, match="scales"):
        B.BlockFP8(codes, torch.ones(3, 10))
    with pytest.raises(ValueError, match="Expected codes"):
        B.BlockFP8(codes[0], scales(3, 10))
    q = B.BlockFP8(codes, scales(3, 10))
    for name, value in (("codes", codes[:5]), ("scales", scales(3, 5)), ("rows", 128)):
        with pytest.raises(AttributeError):
            setattr(q, name, value)


def test_quantize_refusals():
    x = torch.zeros(4, 8)
    for call, error, text in (
            (lambda: B.quantize(x), ValueError, "CUDA tensors"),
            (lambda: B.quantize(x.double()), TypeError, "float32"),
            (lambda: B.quantize(x.long()), TypeError, "float32"),
            (lambda: B.quantize(x[0]), ValueError, "Expected values"),
            (lambda: B.quantize(x[:, :0]), ValueError, "Expected values"),
            (lambda: B.quantize(x, rows=2), ValueError, "1 or 128"),
            (lambda: B.quantize(x, dtype=torch.float16), TypeError, "codes"),
            (lambda: B.quantize_both(x), ValueError, "CUDA tensors")):
        with pytest.raises(error, match=text):
            call()


def test_product_refusals():
    x, w = torch.zeros(4, 256), torch.zeros(8, 256)
    a, b = blocks(4, 256), blocks(8, 256, 128)
    for call, error, text in (
            (lambda: B.matmul(x, b), TypeError, "BlockFP8"),
            (lambda: B.matmul(a, blocks(8, 128)), ValueError, "Expected operands"),
            (lambda: B.matmul(a, blocks(8, 256, lead=(2,))), ValueError, "Expected operands"),
            (lambda: B.matmul(a, b, dtype=torch.float64), TypeError, "matmul gives"),
            (lambda: B.matmul(a, b, bias=torch.zeros(4)), ValueError, "bias"),
            (lambda: B.matmul(a, b, bias=torch.zeros(8).double()), TypeError, "bias"),
            (lambda: B.matmul(a, b), ValueError, "CUDA tensors"),
            (lambda: B.linear(x, w), ValueError, "CUDA tensors"),
            (lambda: B.linear(x, b), ValueError, "CUDA tensors"),
            (lambda: B.linear(x.double(), w), TypeError, "linear takes"),
            (lambda: B.linear(x, w.double()), TypeError, "weight must"),
            (lambda: B.linear(x, w[:, :128]), ValueError, "Expected x"),
            (lambda: B.linear(x, w[:0]), ValueError, "Expected x"),
            (lambda: B.linear(x, w[0]), ValueError, "Expected x"),
            (lambda: B.linear(x, w, torch.zeros(9)), ValueError, "bias"),
            (lambda: B.linear(x, w, grad_dtype=torch.float16), TypeError, "grad_dtype")):
        with pytest.raises(error, match=text):
            call()


def test_grouped_refusals():
    x, w, off = torch.zeros(6, 16).half(), torch.zeros(2, 8, 16).half(), torch.zeros(3, dtype=torch.int32)
    q, wq = blocks(6, 16), blocks(8, 16, 128, lead=(2,))
    out = torch.zeros(6, 8).half()
    for call, error, text in (
            (lambda: grouped_matmul(x, w, off), ValueError, "CUDA tensors"),
            (lambda: grouped_matmul(q, w, off), TypeError, "BlockFP8 weights"),
            (lambda: grouped_matmul(x.float(), w.float(), off), TypeError, "float16 or bfloat16"),
            (lambda: grouped_matmul(x.bfloat16(), w, off), TypeError, "float16 or bfloat16"),
            (lambda: grouped_matmul(x.double(), wq, off), TypeError, "x must be"),
            (lambda: grouped_matmul(x, w[0], off), ValueError, "Expected x"),
            (lambda: grouped_matmul(x[:, :8], w, off), ValueError, "Expected x"),
            (lambda: grouped_matmul(x, w[:, :0], off), ValueError, "Expected x"),
            (lambda: grouped_matmul(x, w.expand(2, 8, 16).repeat(MAX_GROUPS, 1, 1), off), ValueError, "at most 1024"),
            (lambda: grouped_matmul(x, w, off.long()), ValueError, "offsets int32"),
            (lambda: grouped_matmul(x, w, off[:2]), ValueError, "offsets int32"),
            (lambda: grouped_matmul(x, w, off, dtype=torch.float16), ValueError, "dtype is for"),
            (lambda: grouped_matmul(q, wq, off, dtype=torch.float64), TypeError, "the result is"),
            (lambda: grouped_matmul(x, w, off, out=out.float()), ValueError, "Expected out"),
            (lambda: grouped_matmul(x, w, off, out=out.t().contiguous().t()), ValueError, "Expected out"),
            (lambda: grouped_matmul(x, w, off, out=out[:5]), ValueError, "Expected out")):
        with pytest.raises(error, match=text):
            call()


def test_row_strides():
    t = torch.zeros(6, 20)
    assert mx.row_stride(t) == 20 and mx.row_stride(t[:, :7]) == 20 and mx.row_stride(t[::2]) == 40
    assert mx.row_stride(t.t()) is None and mx.row_stride(t[:, ::2]) is None and mx.row_stride(t[:1].expand(6, 20)) is None
    assert mx.row_stride(t[:1, 3:9]) == 6 and mx.row_stride(t[:, :1]) == 20
    b = torch.zeros(3, 6, 20)
    assert mx.row_stride(b) == 20 and mx.row_stride(b[:1].expand(3, 6, 20)) is None
    assert mx.row_stride(b.transpose(0, 1)) is None      # rows of one matrix lie between those of the next


MATRIX = dict(data=4096, scales=64, type=3, rows=8, cols=64, batch=1, ld=64, batch_stride=0, block_rows=1, transposed=0)
HALF = dict(type=2, scales=0, block_rows=0)


def packed(**kw):
    return _lib.MATRIX.pack(*{**MATRIX, **kw}.values())


@pytest.mark.parametrize("a, text", [
    (dict(data=0), "null"), (dict(rows=0), "sizes"), (dict(ld=32), "overlap"), (dict(ld=72), "16-byte"),
    (dict(data=4098), "16-byte"), (dict(type=0), "come with scales"), (dict(type=2), "come with scales"),
    (dict(type=9), "come with scales"), (dict(scales=0), "come with scales"), (HALF, "come with scales"),
    (dict(block_rows=5), "1 or 128"), (dict(cols=128, ld=128), "contraction"), (dict(transposed=1), "row by row"),
    (dict(batch=2, batch_stride=512), "contraction"),
])
def test_c_product_refuses_bad_operands(lib, a, text):
    out = packed(cols=8, ld=8, **HALF)
    status = lib.aeisu_product(packed(**a), packed(), None, 0, out, None, 0, 0, None)
    assert status == _lib.INVALID_ARG and text in _lib.last_error()


def test_c_entries_refuse_bad_arguments(lib):
    codes, half, out = packed(), packed(**HALF), packed(cols=8, ld=8, **HALF)
    f32 = packed(**{**HALF, "type": 0})
    for call, text in (
            (lambda: lib.aeisu_product(None, codes, None, 0, out, None, 0, 0, None), "null"),
            (lambda: lib.aeisu_product(codes, codes, None, 0, None, None, 0, 0, None), "null"),
            (lambda: lib.aeisu_product(codes, codes, 4096, 7, out, None, 0, 0, None), "bias"),
            (lambda: lib.aeisu_product(codes, codes, None, 0, packed(cols=8, ld=4, **HALF), None, 0, 0, None), "output"),
            (lambda: lib.aeisu_product(codes, codes, None, 0, packed(), None, 0, 0, None), "output"),
            (lambda: lib.aeisu_block_quantize(f32, 64, codes, None, 0, None), "1 or 128"),
            (lambda: lib.aeisu_block_quantize(f32, 1, None, None, 0, None), "null"),
            (lambda: lib.aeisu_block_quantize(f32, 1, packed(type=2), None, 0, None), "E4M3"),
            (lambda: lib.aeisu_block_quantize(f32, 1, packed(ld=72), None, 0, None), "16-byte"),
            (lambda: lib.aeisu_block_quantize(f32, 1, packed(rows=9), None, 0, None), "sizes"),
            (lambda: lib.aeisu_block_quantize(f32, 1, codes, codes, 0, None), "transposed sizes"),
            (lambda: lib.aeisu_linear(half, half, None, 0, out, 4096, 1 << 20, 0, None), "scales"),
            (lambda: lib.aeisu_linear(packed(cols=32, **HALF), codes, None, 0, out, 4096, 1 << 20, 0, None), "contraction"),
            (lambda: lib.aeisu_grouped_product(half, half, None, 1, out, 0, None), "offsets"),
            (lambda: lib.aeisu_grouped_product(half, packed(batch=1025, batch_stride=512, **HALF), 4096, 1, out, 0, None), "1024"),
            (lambda: lib.aeisu_grouped_product(half, codes, 4096, 1, out, 0, None), "go together"),
            (lambda: lib.aeisu_grouped_product(half, packed(**{**HALF, "type": 1}), 4096, 1, out, 0, None), "go together"),
            (lambda: lib.aeisu_grouped_product(packed(transposed=1, **HALF), half, 4096, 1, out, 0, None), "contraction"),
            (lambda: lib.aeisu_grouped_weight_gradient(codes, half, 4096, 2, 4096, 2, 0, None), "come with scales"),
            (lambda: lib.aeisu_grouped_weight_gradient(half, packed(rows=9, **HALF), 4096, 2, 4096, 2, 0, None), "contraction"),
            (lambda: lib.aeisu_grouped_weight_gradient(half, half, 4096, 0, 4096, 2, 0, None), "offsets"),
            (lambda: lib.aeisu_grouped_weight_gradient(half, half, 4096, 2, None, 2, 0, None), "output"),
            (lambda: lib.aeisu_column_sum(half, 4096, 2, None, 0, 0, None), "workspace"),
            (lambda: lib.aeisu_product_status(0, None), "null")):
        assert call() == _lib.INVALID_ARG and text in _lib.last_error(), _lib.last_error()
    assert lib.aeisu_linear_kept_bytes(0, 4, 1) == 0 and lib.aeisu_linear_kept_bytes(4, 4, 2) == 0


def test_matrix_layout_matches_the_header(lib):
    class Matrix(C.Structure):
        _fields_ = [("data", C.c_void_p), ("scales", C.c_void_p), ("type", C.c_int), ("rows", C.c_int), ("cols", C.c_int),
                    ("batch", C.c_int), ("ld", C.c_int64), ("batch_stride", C.c_int64), ("block_rows", C.c_int),
                    ("transposed", C.c_int)]
    assert C.sizeof(Matrix) == _lib.MATRIX.size
    m = Matrix.from_buffer_copy(packed(data=1, scales=2, type=3, rows=4, cols=5, batch=6, ld=7, batch_stride=8, block_rows=9,
                                       transposed=10))
    assert [getattr(m, f) for f, _ in Matrix._fields_] == list(range(1, 11))


def test_c_entries_refuse_what_leads_out_of_the_tensors(lib):
    most = 2 ** 31 - 1
    codes, half, out = packed(), packed(**HALF), packed(cols=8, ld=8, **HALF)
    deep = packed(rows=most, ld=64, **HALF)
    for call, text in (
            (lambda: lib.aeisu_product(packed(rows=most), codes, None, 0, packed(rows=most, cols=8, ld=8, **HALF), None, 0, 0, None),
             "sizes"),
            (lambda: lib.aeisu_product(codes, codes, None, 0, packed(rows=7, cols=8, ld=8, **HALF), None, 0, 0, None), "output"),
            (lambda: lib.aeisu_product(codes, codes, None, 0, packed(cols=7, ld=8, **HALF), None, 0, 0, None), "output"),
            (lambda: lib.aeisu_product(codes, codes, None, 0, packed(data=4097, cols=8, ld=8, **HALF), None, 0, 0, None),
             "misaligned"),
            (lambda: lib.aeisu_product(codes, codes, 4098, 0, out, None, 0, 0, None), "misaligned"),
            (lambda: lib.aeisu_block_quantize(deep, 1, packed(rows=most), None, 0, None), "sizes"),
            (lambda: lib.aeisu_block_quantize(packed(data=4097, **HALF), 1, codes, None, 0, None), "misaligned"),
            (lambda: lib.aeisu_block_quantize(half, 1, packed(block_rows=128), None, 0, None), "sizes"),
            (lambda: lib.aeisu_column_sum(deep, 4096, 2, 4096, 1 << 40, 0, None), "sizes"),
            (lambda: lib.aeisu_linear(packed(batch=2, batch_stride=512, **HALF), codes, None, 0, out, 4096, 1 << 20, 0, None), "single"),
            (lambda: lib.aeisu_linear(half, codes, None, 0, packed(rows=9, cols=8, ld=8, **HALF), 4096, 1 << 20, 0, None), "output"),
            (lambda: lib.aeisu_linear_forward(half, packed(batch=2, batch_stride=512, **HALF), None, 0, out, None, None, 4096,
                                              1 << 20, 0, None), "single"),
            (lambda: lib.aeisu_linear_backward(packed(batch=2, batch_stride=512, **HALF), 8, 3, None, None, None, 2, None, 2, None,
                                               2, 4096, 1 << 20, 0, None), "single"),
            (lambda: lib.aeisu_grouped_linear(packed(batch=2, batch_stride=512, **HALF), codes, 4096, 1, out, 4096, 1 << 20, 0,
                                              None), "single"),
            (lambda: lib.aeisu_grouped_product(half, half, 4096, 1, packed(rows=4, cols=8, ld=8, **HALF), 0, None), "output")):
        assert call() == _lib.INVALID_ARG and text in _lib.last_error(), _lib.last_error()
    assert lib.aeisu_linear_kept_bytes(most, 4, 1) == 0 and lib.aeisu_column_sum_workspace(most, 4) == 0
    assert lib.aeisu_grouped_linear_workspace(4, most) == 0 and lib.aeisu_product_workspace(most, 4, 4, 0) == 0
