"""Block-scaled FP8 quantisation, products and the linear layer (aeisu_b200.block_fp8) against the
plain 64-bit forms of tests/block_oracle.py.  Codes and scales are compared bit for bit; products
within the bounds derived there."""
import ctypes as C

import pytest
import torch

import block_oracle as O
from aeisu_b200 import _lib, block_fp8 as B

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    code = C.c_int(-1)
    _lib.check(_lib.lib().aeisu_product_status(0, C.byref(code)))
    assert code.value == 0

E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
HALVES = [torch.bfloat16, torch.float16]


def randn(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed * 7919 + sum(shape))
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def check_codes(q, x, rows, dtype):
    v, s = O.quantize(x, rows, dtype)
    assert q.codes.dtype == dtype and tuple(q.codes.shape) == tuple(x.shape)
    assert torch.equal(q.scales.cpu().double(), s.t())
    assert torch.equal(q.codes.cpu().double().nan_to_num(1e9), v.nan_to_num(1e9))


@pytest.mark.parametrize("m, k", [(1, 1), (1, 128), (3, 129), (33, 16), (130, 257), (127, 520), (257, 1000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 128])
def test_quantize(m, k, dtype, rows):
    x = randn(m, k, dtype=dtype) * torch.exp2(torch.randint(-6, 7, (m, 1))).cuda().to(dtype)
    for codes in (E4, E5):
        check_codes(B.quantize(x, rows=rows, dtype=codes), x, rows, codes)
        q, t = B.quantize_both(x, rows=rows, dtype=codes)
        check_codes(q, x, rows, codes)
        check_codes(t, x.t(), rows, codes)


@pytest.mark.parametrize("m, k, dtype, codes", [
    (57_000, 64, torch.bfloat16, E4), (57_100, 37, torch.float32, E4), (56_961, 8, torch.float16, E5)])
def test_quantize_many_narrow_rows(m, k, dtype, codes):
    # both row blocks of a CTA's 256 rows, with their special values in the first, the second and the last, half a block
    x = randn(m, k + 3, dtype=dtype)[:, 2:k + 2] * torch.exp2(torch.randint(-6, 7, (m, 1))).cuda().to(dtype)
    for r, v in ((3, float("inf")), (130, float("nan")), (200, -float("inf")), (m - 1, float("inf")), (m - 2, 0.0)):
        x[r, r % k] = v
    x[256:384], x[300] = 0, float("nan")
    q, t = B.quantize_both(x, dtype=codes)
    check_codes(q, x, 1, codes)
    check_codes(t, x.t(), 1, codes)
    q, t = B.quantize_both(x.contiguous(), dtype=codes)     # aligned rows
    check_codes(q, x, 1, codes)
    check_codes(t, x.t(), 1, codes)


def test_gradients_of_a_narrow_layer_over_more_rows():
    x, w = randn(60_011, 40, dtype=torch.float16).requires_grad_(), randn(64, 40, seed=1).requires_grad_()
    b, g = randn(64, seed=2).requires_grad_(), randn(60_011, 64, seed=3, scale=1e-2, dtype=torch.float16)
    y = B.linear(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g)
    rows = torch.arange(0, 60_011, 211)
    O.check_product(y.detach()[rows.cuda()], O.values(x.detach()[rows.cuda()]), O.values(w.detach(), 128), b.detach())
    O.check_product(gx[rows.cuda()], O.values(g[rows.cuda()]), O.values(w.detach().t(), 128))
    O.check_product(gw, O.values(g.t()), O.values(x.detach().t()))
    s = g.double().cpu()
    O.check(gb, s.sum(0), 60_012 * 2.0 ** -24 * s.abs().sum(0))


def test_quantize_batch_and_strides():
    x = randn(3, 130, 200, dtype=torch.bfloat16)
    q = B.quantize(x, rows=128)
    for i in range(3):
        check_codes(B.BlockFP8(q.codes[i], q.scales[i], 128), x[i], 128, E4)
    wide = randn(40, 400)
    for v in (wide[:, 3:300], wide[1::2, ::1], wide.t(), wide[:, ::2], wide[:1].expand(20, 400), wide[5:6, 7:8]):
        check_codes(B.quantize(v), v, 1, E4)
        check_codes(B.quantize_both(v)[1], v.t(), 1, E4)


@pytest.mark.parametrize("codes", [E4, E5])
@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_extremes(codes, rows):
    top = O.TOP[codes][0]
    x = torch.zeros(140, 300)
    x[1, :5] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0, -2.0])   # a block beside NaN
    x[2, 130] = float("inf")                                   # an infinity among zeros
    x[3] = 3.4e38
    x[4, 0], x[4, 1] = 1e-45, -3e-39                           # subnormal
    x[5, 128] = top                                            # the largest code itself
    x[6, 128] = torch.nextafter(torch.tensor(top), torch.tensor(1e9))
    x[7, :128] = torch.linspace(-1, 1, 128) * top
    x[8, 0], x[8, 1] = -0.0, 2.0 ** -140
    x = x.cuda()
    order = [x] if rows == 1 else [x[i:i + 1].expand(4, 300).contiguous() for i in range(9)] + [x]
    for v in order:
        check_codes(B.quantize(v, rows=rows, dtype=codes), v, rows, codes)
        check_codes(B.quantize_both(v, rows=rows, dtype=codes)[1], v.t(), rows, codes)


def test_dequantize():
    x = randn(70, 300)
    for rows in (1, 128):
        assert torch.equal(B.quantize(x, rows=rows).dequantize().cpu().double(), O.values(x, rows))


def random_blocks(r, c, rows, dtype, seed):
    """An operand with scales that differ wildly from block to block, so that one scale read for another shows."""
    g = torch.Generator().manual_seed(seed)
    v = torch.randn(r, c, generator=g).cuda().to(dtype)
    s = torch.randint(117, 138, (-(-c // 128), -(-r // rows)), generator=g).to(torch.uint8).cuda()
    return B.BlockFP8(v, s.view(torch.float8_e8m0fnu), rows)


SIZES = [(1, 1, 1), (1, 16, 128), (1, 300, 4096), (2, 129, 130), (5, 17, 33), (16, 128, 512), (17, 1000, 640),
         (64, 100, 1100), (65, 200, 64), (127, 64, 255), (128, 256, 128), (129, 128, 257), (300, 1000, 520),
         (513, 48, 32), (1030, 333, 700), (2000, 2050, 129), (100, 131, 1100), (200, 77, 4096), (90, 512, 2048)]


@pytest.mark.parametrize("m, n, k", SIZES)
@pytest.mark.parametrize("types", [(E4, E4), (E5, E4)])
def test_matmul(m, n, k, types):
    a, b = random_blocks(m, k, 1, types[0], 1), random_blocks(n, k, 128, types[1], 2)
    O.check_product(B.matmul(a, b, dtype=torch.float32), a.dequantize(), b.dequantize())
    bias = randn(n, scale=100.0)
    O.check_product(B.matmul(a, b, bias=bias), a.dequantize(), b.dequantize(), bias)


@pytest.mark.parametrize("m, n, k", [(64, 128, 20_000), (33, 17, 30_001), (1, 100, 40_000), (130, 120, 25_000)])
def test_long_contractions_in_parts(m, n, k):
    # few outputs: the contraction is cut over all SMs and the parts are joined by a second kernel
    a, b, bias = random_blocks(m, k, 1, E4, 1), random_blocks(n, k, 1, E4, 2), randn(n, scale=1e4)
    for dtype in (torch.float32, torch.bfloat16):
        y = B.matmul(a, b, bias=bias, dtype=dtype)
        O.check_product(y, a.dequantize(), b.dequantize(), bias)
        assert torch.equal(y, B.matmul(a, b, bias=bias, dtype=dtype))


def test_gradients_of_a_narrow_layer_over_many_rows():
    x, w = randn(20_011, 64, dtype=torch.bfloat16).requires_grad_(), randn(48, 64, seed=1, dtype=torch.bfloat16).requires_grad_()
    b, g = randn(48, seed=2).requires_grad_(), randn(20_011, 48, seed=3, scale=1e-3, dtype=torch.bfloat16)
    gx, gw, gb = torch.autograd.grad(B.linear(x, w, b), (x, w, b), g)
    rows = torch.arange(0, 20_011, 97)
    O.check_product(gx[rows.cuda()], O.values(g[rows.cuda()]), O.values(w.detach().t(), 128))
    O.check_product(gw, O.values(g.t()), O.values(x.detach().t()))
    s = g.double().cpu()
    O.check(gb, s.sum(0), 20_012 * 2.0 ** -24 * s.abs().sum(0))


@pytest.mark.parametrize("rows", [(1, 1), (128, 1), (128, 128)])
def test_matmul_block_rows(rows):
    for m, n, k in ((3, 200, 300), (150, 200, 300), (300, 40, 300)):
        a, b = random_blocks(m, k, rows[0], E4, 3), random_blocks(n, k, rows[1], E4, 4)
        O.check_product(B.matmul(a, b, dtype=torch.float16), a.dequantize(), b.dequantize())


def test_matmul_is_exact_on_small_integers():
    # Integers up to 8 with scale 1: every product and sum is an integer below 2^24, so the result is exact.
    g = torch.Generator().manual_seed(5)
    for m, n, k in ((1, 512, 2048), (200, 300, 2048), (700, 520, 1024)):
        a, b = (torch.randint(-8, 9, (r, k), generator=g).float().cuda() for r in (m, n))
        ones = lambda r: torch.full((-(-k // 128), r), 127, dtype=torch.uint8).cuda().view(torch.float8_e8m0fnu)  # noqa: E731
        y = B.matmul(B.BlockFP8(a.to(E4), ones(m)), B.BlockFP8(b.to(E4), ones(n)), dtype=torch.float32)
        assert torch.equal(y.double(), a.double() @ b.double().t())


def test_matmul_confines_nan():
    x, w = randn(70, 300), randn(90, 300)
    x[3, 200] = float("nan")
    x[69, 0] = float("inf")
    w[5, 299] = float("-inf")
    y = B.matmul(B.quantize(x), B.quantize(w), dtype=torch.float32)
    O.check_product(y, O.values(x), O.values(w))
    assert bool(y[3].isnan().all() and y[:, 5].isnan().all()) and int(y.isnan().sum()) == 2 * 90 + 70 - 2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m, k, n, bias", [(1, 128, 64, True), (5, 40, 33, False), (300, 130, 70, True),
                                           (1025, 512, 384, True), (70, 1024, 1000, False)])
def test_linear_gradients(dtype, m, k, n, bias):
    x = randn(m, k, dtype=dtype).requires_grad_()
    w = randn(n, k, seed=1, scale=k ** -0.5, dtype=dtype).requires_grad_()
    b = randn(n, seed=2, dtype=dtype).requires_grad_() if bias else None
    g = randn(m, n, seed=3, scale=1e-2, dtype=dtype)
    y = B.linear(x, w, b)
    y.backward(g)
    assert y.dtype == dtype and x.grad.dtype == dtype and w.grad.dtype == dtype
    xd, wd = x.detach(), w.detach()
    O.check_product(y, O.values(xd), O.values(wd, 128), None if b is None else b.detach())
    O.check_product(x.grad, O.values(g), O.values(wd.t(), 128))
    O.check_product(w.grad, O.values(g.t()), O.values(xd.t()))
    if b is not None:
        s = g.double().cpu()
        O.check(b.grad, s.sum(0), (m + 1) * 2.0 ** -24 * s.abs().sum(0) + O.half_step(s.sum(0).abs() * (1 + 2 ** -10), dtype))


def test_linear_gradient_against_differences():
    # The layer is linear in what the quantised input stands for: moving one input by a whole code step
    # moves the loss by the step times the gradient of the exact layer, which the FP8 gradient equals
    # up to the rounding of g (2^-4 relative to each value).
    x, w = randn(4, 128, dtype=torch.float32).round().clamp(-4, 4), randn(32, 128, seed=1)
    x[:, 0] = 8.0   # the block maximum: codes are integers, the scale does not move
    g = torch.randint(-4, 5, (4, 32)).float().cuda()
    g[:, 0] = 8.0   # exact in E4M3, so the gradient is too
    xr = x.clone().requires_grad_()
    B.linear(xr, w).backward(g)
    for r, c in ((0, 5), (1, 77), (3, 127)):
        up, down = x.clone(), x.clone()
        up[r, c] += 1.0
        down[r, c] -= 1.0
        with torch.no_grad():
            d = ((B.linear(up, w) - B.linear(down, w)).double() * g.double()).sum() / 2
        # float32 sums of 128 and 32 terms of size |w| <= 5
        assert abs(float(d) - float(xr.grad[r, c])) < 160 * 2.0 ** -23 * 5 * 8 * 32


@pytest.mark.parametrize("wants", [(True, False), (False, True)])
def test_linear_partial_gradients_and_shapes(wants):
    x = randn(2, 5, 9, 64, dtype=torch.bfloat16).requires_grad_(wants[0])
    w = randn(48, 64, seed=1, dtype=torch.bfloat16).requires_grad_(wants[1])
    y = B.linear(x, w)
    assert tuple(y.shape) == (2, 5, 9, 48)
    y.sum().backward()          # an expanded gradient without strides
    g = torch.ones(90, 48)
    assert (x.grad is not None) == wants[0] and (w.grad is not None) == wants[1]
    if wants[0]:
        O.check_product(x.grad.reshape(90, 64), O.values(g), O.values(w.detach().t(), 128))
    if wants[1]:
        O.check_product(w.grad, O.values(g.t()), O.values(x.detach().reshape(90, 64).t()))


def test_linear_serving_matches_training_forward():
    x, w, b = randn(7, 200, dtype=torch.float16), randn(130, 200, seed=1, dtype=torch.float16), randn(130, seed=2)
    kept = B.quantize(w, rows=128)
    y = B.linear(x, kept, b)
    assert torch.equal(y, B.linear(x, w, b))
    assert torch.equal(y, B.linear(x, w.clone().requires_grad_(), b).detach())
    assert torch.equal(y, B.matmul(B.quantize(x), kept, bias=b, dtype=torch.float16))


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17])
@pytest.mark.parametrize("n, k", [(17, 8), (130, 200), (1000, 4096), (257, 1032), (64, 130)])
def test_few_rows_are_quantised_alike(m, n, k):
    # few aligned 16-bit rows are quantised inside the product, others by a kernel of their own: the same codes, so
    # the same bits, whatever the rows hold
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = randn(m, k, dtype=dtype) * torch.exp2(torch.arange(m).float() - 8)[:, None].cuda().to(dtype)
        w, b = B.quantize(randn(n, k, seed=1), rows=128), randn(n, seed=2)
        if m > 4:
            x[1], x[2, 0], x[3, k // 2:], x[4, -1] = 0, float("nan"), float("inf"), -float("inf")
        for v in (x, torch.nn.functional.pad(x, (1, 8))[:, 1:k + 1]):
            y = B.linear(v, w, b)
            assert torch.equal(y.nan_to_num(1e9), B.matmul(B.quantize(v), w, bias=b, dtype=dtype).nan_to_num(1e9))
        if m <= 4:
            O.check_product(y, O.values(x), w.dequantize(), b)


def test_linear_empty():
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = randn(32, 64, dtype=torch.bfloat16).requires_grad_()
    b = randn(32, dtype=torch.bfloat16).requires_grad_()
    y = B.linear(x, w, b)
    assert tuple(y.shape) == (0, 32)
    y.sum().backward()
    assert tuple(x.grad.shape) == (0, 64) and not w.grad.any() and not b.grad.any()
    q = B.quantize(x)
    assert tuple(q.codes.shape) == (0, 64) and tuple(q.scales.shape) == (1, 0)
    assert tuple(B.matmul(q, B.quantize(w, rows=128)).shape) == (0, 32)


def test_operands_without_alignment():
    # codes whose rows start anywhere: the product takes a copy
    a, b = random_blocks(20, 77, 1, E4, 1), random_blocks(40, 77, 128, E4, 2)
    raw = torch.zeros(20 * 81 + 3, dtype=torch.uint8, device="cuda")
    codes = raw[3:].as_strided((20, 77), (81, 1), 3).view(E4)
    codes.view(torch.uint8).copy_(a.codes.contiguous().view(torch.uint8))
    want = B.matmul(a, b)
    assert torch.equal(B.matmul(B.BlockFP8(codes, a.scales), b), want)
    tall = a.codes.t().contiguous().t()     # stored column by column
    assert torch.equal(B.matmul(B.BlockFP8(tall, a.scales), b), want)


def test_stream_device_and_repeats():
    x, w = randn(300, 520, dtype=torch.bfloat16), randn(200, 520, seed=1, dtype=torch.bfloat16)
    want = B.linear(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [B.linear(x, w) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(v, want) for v in got)


def test_graph_capture_replays_with_new_inputs():
    x = randn(3, 256, dtype=torch.bfloat16)
    w = B.quantize(randn(512, 256, seed=1), rows=128)
    xt = randn(40, 64, seed=5, dtype=torch.bfloat16).requires_grad_()
    wt = randn(48, 64, seed=6, dtype=torch.bfloat16).requires_grad_()

    def step():
        y = B.linear(x, w)
        return y, *torch.autograd.grad(B.linear(xt, wt).square().sum(), (xt, wt))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (7, 8):
        with torch.no_grad():
            x.copy_(randn(3, 256, seed=seed))
            xt.copy_(randn(40, 64, seed=seed))
        graph.replay()
        want = step()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_linear_mixed_types_and_strides():
    # activations in bfloat16 with a float32 master weight and a strided bias, everything a view
    x = randn(70, 300, dtype=torch.bfloat16)[:, 3:203].requires_grad_()
    w = randn(200, 130, seed=1).t().requires_grad_()
    b = randn(260, seed=2)[::2].requires_grad_()
    g = randn(130, 70, seed=3).bfloat16().t()
    y = B.linear(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g)
    assert y.dtype == gx.dtype == torch.bfloat16 and gw.dtype == gb.dtype == torch.float32
    O.check_product(y, O.values(x.detach()), O.values(w.detach(), 128), b.detach())
    O.check_product(gx, O.values(g), O.values(w.detach().t(), 128))
    O.check_product(gw, O.values(g.t()), O.values(x.detach().t()))
    assert torch.equal(gb, torch.autograd.grad(B.linear(x, w, b), b, g)[0])


def test_linear_e5m2_gradients():
    x, w = (randn(*s, seed=i).requires_grad_() for i, s in enumerate(((150, 96), (72, 96))))
    g = randn(150, 72, seed=2) * torch.exp2(torch.randint(-20, 20, (150, 1), generator=torch.Generator().manual_seed(0))).cuda()
    gx, gw = torch.autograd.grad(B.linear(x, w, grad_dtype=E5), (x, w), g)
    O.check_product(gx, O.values(g, dtype=E5), O.values(w.detach().t(), 128))
    O.check_product(gw, O.values(g.t(), dtype=E5), O.values(x.detach().t()))


def test_infinite_gradients_reach_the_bias_as_they_are():
    x, w, b = randn(200, 64), randn(32, 64, seed=1).requires_grad_(), randn(32, seed=2).requires_grad_()
    g = randn(200, 32, seed=3)
    g[7, 3], g[150, 4], g[1, 5], g[2, 5] = float("inf"), float("nan"), float("inf"), -float("inf")
    gw, gb = torch.autograd.grad(B.linear(x, w, b), (w, b), g)
    assert torch.equal(gb.isnan(), g.sum(0).isnan()) and torch.equal(gb.isinf(), g.sum(0).isinf())
    assert torch.equal(gw.isnan().any(1), torch.isin(torch.arange(32), torch.tensor([3, 4, 5])).cuda())


def test_more_than_two_to_the_31_elements():
    rows, k = 270_000, 8192
    x = torch.empty(rows, k, device="cuda", dtype=torch.bfloat16).normal_(generator=torch.Generator("cuda").manual_seed(1))
    w = B.quantize(randn(24, k, seed=2), rows=128)
    q, t = B.quantize_both(x)
    ends = (slice(0, 100), slice(rows - 100, rows))
    for s in ends:
        part = B.quantize(x[s])
        assert torch.equal(q.codes[s].view(torch.uint8), part.codes.view(torch.uint8))
        assert torch.equal(q.scales[:, s].view(torch.uint8), part.scales.view(torch.uint8))
    last = x[rows // 128 * 128:]        # the last block of the transpose, which starts on a multiple of 128
    lt = B.quantize(last.t())
    assert torch.equal(t.codes[:, rows // 128 * 128:].view(torch.uint8), lt.codes.view(torch.uint8))
    assert torch.equal(t.scales[-1].view(torch.uint8), lt.scales[0].view(torch.uint8))
    y = B.matmul(q, w, dtype=torch.float32)
    for s in ends:
        O.check_product(y[s], q.codes[s].double().cpu() * q.scales[:, s].float().t().repeat_interleave(128, 1).double().cpu(),
                        w.dequantize())


def test_two_streams_at_once():
    a, b = randn(1500, 1024, dtype=torch.bfloat16), randn(900, 2048, seed=1, dtype=torch.bfloat16)
    wa, wb = randn(700, 1024, seed=2, dtype=torch.bfloat16), randn(512, 2048, seed=3, dtype=torch.bfloat16)
    want = B.linear(a, wa), B.linear(b, wb)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = [], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for s, x, w, o in ((streams[0], a, wa, got[0]), (streams[1], b, wb, got[1])):
            with torch.cuda.stream(s):
                o.append(B.linear(x, w))
    torch.cuda.synchronize()
    for o, w in zip(got, want):
        assert all(torch.equal(v, w) for v in o)


def test_refusals_on_the_gpu():
    x, w = randn(4, 64, dtype=torch.bfloat16), randn(32, 64, seed=1, dtype=torch.bfloat16)
    kept = B.quantize(w, rows=128)
    with pytest.raises(ValueError, match="without gradients"):
        B.linear(x.requires_grad_(), kept)
    with pytest.raises(ValueError, match="CUDA tensors"):
        B.linear(x, w.cpu())
    with pytest.raises(ValueError, match="bias"):
        B.linear(x, w, randn(31))
    with pytest.raises(RuntimeError):
        v = randn(4, 64).requires_grad_()
        (g,) = torch.autograd.grad(B.linear(v, w).sum(), v, create_graph=True)
        g.sum().backward()
