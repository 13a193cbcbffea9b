"""Block-scaled FP8 and grouped products at the edges of what they promise: operands quantised by the kernel
just before, exact sums over many rows, the largest contractions and outputs, the state of bounded waits."""
import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad

from aeisu_b200 import _lib, block_fp8 as B
from aeisu_b200.grouped import grouped_matmul

pytestmark = pytest.mark.gpu
E4 = torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    code = C.c_int(-1)
    _lib.check(_lib.lib().aeisu_product_status(0, C.byref(code)))
    assert code.value == 0


def randn(*shape, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed * 7919 + sum(shape))
    return torch.randn(shape, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("m, k, n", [(40, 512, 384), (300, 1024, 640), (2000, 256, 512)])
def test_products_read_the_scales_of_this_call(m, k, n):
    # The product starts while the quantiser writes its operand's scales, into memory that the call before used: with
    # inputs that differ by powers of two from call to call, a scale read too early is that of another call.
    kept, off = B.quantize(randn(n, k, seed=1), rows=128), torch.tensor([0, m // 3, m], dtype=torch.int32).cuda()
    experts = B.quantize(randn(2, n, k, seed=2), rows=128)
    inputs = [randn(m, k) * 2.0 ** e * torch.exp2(torch.arange(m).cuda() % 5 - 2)[:, None].bfloat16() for e in (0, 9, -7)]
    coded = [B.quantize(x) for x in inputs]
    want = [(B.matmul(q, kept), grouped_matmul(q, experts, off)) for q in coded]
    w, g = randn(n, k, seed=3).requires_grad_(), randn(m, n, seed=4)
    grads = [torch.autograd.grad(B.linear(x, w), w, g)[0] for x in inputs]
    torch.cuda.synchronize()
    for _ in range(20):
        out = [(B.linear(x, kept), grouped_matmul(x, experts, off), *torch.autograd.grad(B.linear(x, w), w, g))
               for x in inputs]
        for got, (y, z), gw in zip(out, want, grads):
            assert torch.equal(got[0], y) and torch.equal(got[1], z) and torch.equal(got[2], gw)


@pytest.mark.parametrize("k", [2 ** 31 - 1025, 2 ** 31 - 12_000])
def test_longest_contraction(k):
    # 148 parts, the last of which would end beyond 2^31 if it were as long as the others: ones at both ends and around
    # the middle, so that every product and sum is a whole number below 2^24
    codes = torch.zeros(1, k, dtype=torch.uint8, device="cuda")
    codes[:, :70_000] = 0x38                      # 1.0
    codes[:, k // 2:k // 2 + 300] = 0x40          # 2.0
    codes[:, -90_001:] = 0x38
    scales = torch.full((-(-k // 128), 1), 127, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    a = B.BlockFP8(codes.view(E4), scales)
    got = float(B.matmul(a, a, dtype=torch.float32))
    assert got == 70_000 + 4 * 300 + 90_001


def unit_blocks(*shape, rows=1):
    """An operand of ones."""
    codes = torch.full(shape, 0x38, dtype=torch.uint8, device="cuda").view(E4)
    lead, (r, c) = shape[:-2], shape[-2:]
    scales = torch.full((*lead, -(-c // 128), -(-r // rows)), 127, dtype=torch.uint8, device="cuda")
    return B.BlockFP8(codes, scales.view(torch.float8_e8m0fnu), rows)


def used_memory(n, dtype):
    """Leaves n elements of memory full of threes to the next allocation of their size."""
    torch.full((n,), 3.0, device="cuda", dtype=dtype)


def test_rows_in_no_group_of_more_than_two_to_the_31_bytes():
    n = 2 ** 29
    x, w = unit_blocks(3, 16), unit_blocks(1, n, 16, rows=128)
    used_memory(3 * n, torch.float32)
    y = grouped_matmul(x, w, torch.tensor([1, 2], dtype=torch.int32).cuda(), dtype=torch.float32)
    seen = [float(f(r)) for r in y for f in (torch.min, torch.max)]    # (a failing assert prints what it names)
    assert seen == [0, 0, 16, 16, 0, 0]


def test_as_many_rows_in_no_group_as_there_may_be():
    # one group of one row: the rows that the warps would take after the last ones lie beyond 2^31
    t = 2 ** 31 - 1025
    codes = torch.empty(t, 16, dtype=torch.uint8, device="cuda")
    codes[:2] = 0x38
    scales = torch.full((1, t), 127, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    x, w = B.BlockFP8(codes.view(E4)[:, :1], scales), unit_blocks(1, 1, 1)
    used_memory(t, torch.float16)
    y = grouped_matmul(x, w, torch.tensor([1, 2], dtype=torch.int32).cuda(), dtype=torch.float16)
    seen = float(y[0]), float(y[1]), bool(y[2:].any())
    assert seen == (0, 1, False)


def test_weight_gradient_that_takes_more_than_two_seconds():
    # One tile whose 8,281,251 steps take about 4.4e9 cycles: every wait that spans them has to last as long, that for
    # the last, partial step too.  Ones among zeros, so that the sums are exact.
    t = 530_000_005
    x, g = (torch.zeros(t, 8, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    for i, r in enumerate((0, 63, 1_000_001, t - 6, t - 5, t - 1)):
        x[r, i], g[r, i] = 1 + i, 2
    w = torch.zeros(1, 8, 8, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = grouped_matmul(x, w, torch.tensor([0, t], dtype=torch.int32).cuda())
    (gw,) = torch.autograd.grad(y, w, g)
    assert gw[0].tolist() == torch.diag(torch.tensor([2.0, 4, 6, 8, 10, 12, 0, 0])).tolist()


def test_tangents_of_gradients_are_refused():
    x, off = randn(8, 64), torch.tensor([0, 3, 8], dtype=torch.int32).cuda()
    w, we = randn(32, 64, seed=1).requires_grad_(), randn(2, 32, 64, seed=2).requires_grad_()
    for y, leaf in ((B.linear(x, w), w), (grouped_matmul(x, we, off), we)):
        with forward_ad.dual_level():
            g = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(ValueError, match="forward-mode"):
                torch.autograd.grad(y, leaf, g, retain_graph=True)
            assert torch.autograd.grad(y, leaf, torch.ones_like(y))[0].isfinite().all()


def test_check_products_after_products():
    for device in (None, 0, "cuda", torch.device("cuda", 0)):
        B.matmul(unit_blocks(300, 640), unit_blocks(200, 640, rows=128))
        assert B.check_products(device) is None


def test_views_of_negated_memory():
    # the imaginary part of a conjugate: its memory holds the values with the other sign
    def imaginary(*shape, seed, dtype=torch.float32):
        z = torch.view_as_complex(randn(*shape, 2, seed=seed, dtype=dtype)).conj().imag
        assert z.is_neg()
        return z, z.resolve_neg().clone()

    off = torch.tensor([0, 3, 5], dtype=torch.int32).cuda()
    for rows, cols in ((5, 1), (1, 1), (5, 40)):
        x, x0 = imaginary(rows, cols, seed=1)
        w, w0 = imaginary(24, cols, seed=2)
        b, b0 = imaginary(24, seed=3)
        one, one0 = imaginary(1, seed=4)
        kept = B.quantize(w0, rows=128)
        assert torch.equal(B.quantize(x).dequantize(), B.quantize(x0).dequantize())
        assert torch.equal(B.linear(x, kept, b), B.linear(x0, kept, b0))
        assert torch.equal(B.linear(x, w, b), B.linear(x0, w0, b0))
        assert torch.equal(B.linear(x, w[:1], one), B.linear(x0, w0[:1], one0))
        g, g0 = imaginary(rows, 24, seed=5)
        leaf = w0.clone().requires_grad_()
        grads = [torch.autograd.grad(B.linear(x0, leaf), leaf, v)[0] for v in (g, g0)]
        assert torch.equal(*grads)
        experts = B.quantize(torch.stack([w0, w0]), rows=128)
        assert torch.equal(grouped_matmul(x, experts, off), grouped_matmul(x0, experts, off))
        half, half0 = imaginary(rows, cols, seed=6, dtype=torch.float16)
        we = torch.stack([w0, w0]).half()
        assert torch.equal(grouped_matmul(half, we, off), grouped_matmul(half0, we, off))
        out = imaginary(rows, 24, seed=7, dtype=torch.float16)[0]
        with pytest.raises(ValueError, match="Expected out"):
            grouped_matmul(half, we, off, out=out)


def integers(*shape, most, seed, dtype):
    g = torch.Generator().manual_seed(seed * 7919 + sum(shape))
    return torch.randint(-most, most + 1, shape, generator=g).to(dtype).cuda()


@pytest.mark.parametrize("m, k, n, dtype", [
    (60_011, 40, 64, torch.float16), (60_011, 37, 50, torch.bfloat16), (57_217, 8, 24, torch.float32),
    (60_011, 200, 64, torch.bfloat16), (57_100, 64, 130, torch.float16), (20_011, 64, 48, torch.bfloat16)])
def test_sums_over_many_rows_are_whole(m, k, n, dtype):
    # Integers of at most three bits are exact in E4M3 and sums of their products stay below 2^24, so that a row block, a
    # part or a CTA's half that is lost, or counted twice, changes the result.
    x, w = integers(m, k, most=3, seed=1, dtype=dtype).requires_grad_(), integers(n, k, most=3, seed=2, dtype=torch.float32).requires_grad_()
    b, g = integers(n, most=7, seed=3, dtype=torch.float32).requires_grad_(), integers(m, n, most=2, seed=4, dtype=dtype)
    g[:128] = 1                                  # the first block and, below, the last rows do not cancel
    g[-(m % 128 or 128):] = -2
    x0, w0, g0 = (v.detach().double() for v in (x, w, g))
    y = B.linear(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g)
    assert torch.equal(y.detach(), (x0 @ w0.t() + b.detach().double()).to(dtype))
    assert torch.equal(gx, (g0 @ w0).to(dtype))
    assert torch.equal(gw.double(), g0.t() @ x0) and torch.equal(gb.double(), g0.sum(0))
    # infinities and NaN stay in their columns of the bias' and the weight's gradient
    g[m - 1, 1], g[300, 2], g[m // 2, n - 1] = float("inf"), float("nan"), -float("inf")
    y = B.linear(x, w, b)
    gx, gw2, gb2 = torch.autograd.grad(y, (x, w, b), g)
    fine = torch.ones(n, dtype=torch.bool, device="cuda")
    fine[[1, 2, n - 1]] = False
    assert torch.equal(gw2[fine], gw[fine]) and bool(gw2[~fine].isnan().all())
    assert torch.equal(gb2[fine], gb[fine])
    assert float(gb2[1]) == float("inf") and float(gb2[n - 1]) == -float("inf") and bool(gb2[2].isnan())


@pytest.mark.parametrize("m, n, ld", [(1, 1, 1), (63, 64, 64), (1000, 65, 72), (100_003, 37, 40), (130_000, 8, 8), (5, 4000, 4000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_column_sum_entry(m, n, ld, dtype):
    x = integers(m, ld, most=7, seed=m, dtype=dtype)[:, :n]
    types = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    lib = _lib.lib()
    size = lib.aeisu_column_sum_workspace(m, n)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    want = x.double().sum(0)
    for out_type in (torch.float32, torch.bfloat16):
        out = torch.full((n,), 99.0, dtype=out_type, device="cuda")
        mat = _lib.MATRIX.pack(x.data_ptr(), 0, types[dtype], m, n, 1, ld, 0, 0, 0)
        _lib.check(lib.aeisu_column_sum(mat, out.data_ptr(), types[out_type], ws.data_ptr(), size, 0,
                                        torch.cuda.current_stream().cuda_stream))
        assert torch.equal(out, want.to(out_type))
