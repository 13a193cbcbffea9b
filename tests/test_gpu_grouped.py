"""Products grouped by expert (aeisu_b200.grouped) against plain 64-bit loops over the groups."""
import ctypes as C

import pytest
import torch

import block_oracle as O
from aeisu_b200 import _lib, block_fp8 as B
from aeisu_b200.grouped import grouped_matmul

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    code = C.c_int(-1)
    _lib.check(_lib.lib().aeisu_product_status(0, C.byref(code)))
    assert code.value == 0

HALVES = [torch.bfloat16, torch.float16]


def randn(*shape, seed=0, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed * 7919 + sum(shape))
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def bounds(sizes, first=0):
    return torch.tensor([first] + sizes).cumsum(0).to(torch.int32).cuda()


def spans(off):
    v = off.tolist()
    return list(zip(v, v[1:]))


GROUPS = [[1], [128], [5, 0, 3], [0, 0, 7], [130, 1, 0, 127], [64, 200, 300, 2], [0, 1000, 0], [33] * 40,
          [3, 0, 1, 0, 0, 9, 2, 1], [16] * 16, [700, 100]]
WIDTHS = [(8, 8), (64, 64), (200, 76), (33, 17), (256, 384), (520, 130)]


@pytest.mark.parametrize("sizes", GROUPS, ids=str)
@pytest.mark.parametrize("k, n", WIDTHS)
def test_forward_and_gradients(sizes, k, n):
    dtype = HALVES[(k + len(sizes)) % 2]
    t, e = sum(sizes), len(sizes)
    off = bounds(sizes)
    x = randn(t, k, dtype=dtype).requires_grad_()
    w = randn(e, n, k, seed=1, scale=k ** -0.5, dtype=dtype).requires_grad_()
    g = randn(t, n, seed=2, dtype=dtype)
    y = grouped_matmul(x, w, off)
    y.backward(g)
    assert y.dtype == dtype and torch.equal(y.detach(), grouped_matmul(x.detach(), w.detach(), off))
    for i, (lo, hi) in enumerate(spans(off)):
        O.check_product(y[lo:hi], x.detach()[lo:hi], w.detach()[i])
        O.check_product(x.grad[lo:hi], g[lo:hi], w.detach()[i].t())
        O.check_product(w.grad[i], g[lo:hi].t(), x.detach()[lo:hi].t())


@pytest.mark.parametrize("sizes", GROUPS, ids=str)
@pytest.mark.parametrize("k, n", WIDTHS)
def test_fp8_weights(sizes, k, n):
    off, x, w = bounds(sizes), randn(sum(sizes), k), randn(len(sizes), n, k, seed=1)
    kept, q = B.quantize(w, rows=128), B.quantize(x)
    y = grouped_matmul(x, kept, off)
    assert y.dtype == torch.bfloat16 and torch.equal(y, grouped_matmul(q, kept, off))
    exact = grouped_matmul(q, kept, off, dtype=torch.float32)
    xv, wv = q.dequantize(), kept.dequantize()
    for i, (lo, hi) in enumerate(spans(off)):
        O.check_product(y[lo:hi], xv[lo:hi], wv[i])
        O.check_product(exact[lo:hi], xv[lo:hi], wv[i])


@pytest.mark.parametrize("sizes", [[5, 0, 3], [37, 130, 60], [300, 201]], ids=str)
@pytest.mark.parametrize("rows, weight_rows", [(128, 128), (128, 1), (1, 1)])
def test_fp8_operands_of_either_block_height(sizes, rows, weight_rows):
    # a group starts anywhere in a block of 128 rows of x, and its tiles reach into the next
    t, off = sum(sizes) + 11, bounds(sizes, first=11)
    x = B.quantize(randn(t, 300) * torch.exp2(torch.arange(t).float() // 64 - 4)[:, None].cuda(), rows=rows)
    w = B.quantize(randn(len(sizes), 150, 300, seed=1), rows=weight_rows)
    y = grouped_matmul(x, w, off, dtype=torch.float32)
    xv, wv = x.dequantize(), w.dequantize()
    for i, (lo, hi) in enumerate(spans(off)):
        O.check_product(y[lo:hi], xv[lo:hi], wv[i])
    assert not y[:11].any()


def test_gradient_against_differences():
    # The product is linear: a whole step in one entry moves the weighted sum by the gradient exactly,
    # up to float16's rounding of the outputs and of the gradient (integers here: both exact).
    off = bounds([3, 0, 5])
    gen = torch.Generator().manual_seed(3)
    ints = lambda *s: torch.randint(-3, 4, s, generator=gen).half().cuda()  # noqa: E731
    x, w, g = ints(8, 24).requires_grad_(), ints(3, 16, 24).requires_grad_(), ints(8, 16)
    grouped_matmul(x, w, off).backward(g)
    with torch.no_grad():
        loss = lambda a, b: (grouped_matmul(a, b, off).double() * g.double()).sum()  # noqa: E731
        for r, c in ((0, 0), (2, 23), (7, 11)):
            d = torch.zeros_like(x)
            d[r, c] = 1
            assert float((loss(x + d, w) - loss(x - d, w)) / 2) == float(x.grad[r, c])
        for i, r, c in ((0, 0, 0), (1, 3, 3), (2, 15, 23)):
            d = torch.zeros_like(w)
            d[i, r, c] = 1
            assert float((loss(x, w + d) - loss(x, w - d)) / 2) == float(w.grad[i, r, c])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("sizes", [[40, 0, 30], [300, 200]], ids=str)
def test_rows_outside_the_groups(fp8, sizes):
    t = sum(sizes) + 60
    off = bounds(sizes, first=21)        # rows before the first group and behind the last
    x, w = randn(t, 128), randn(len(sizes), 136, 128, seed=1)
    x[:21] = float("nan")                # nobody reads them
    x[int(off[-1]):] = float("inf")
    weight = B.quantize(w, rows=128) if fp8 else w
    y = grouped_matmul(x, weight, off)
    inside = torch.zeros(t, dtype=torch.bool)
    inside[21:int(off[-1])] = True
    assert not y.cpu()[~inside].any() and bool(y.cpu()[inside].isfinite().all())
    out = torch.full((t, 136), 7.0, device="cuda", dtype=torch.bfloat16)
    assert grouped_matmul(x, weight, off, out=out) is out
    assert bool((out.cpu()[~inside] == 7).all()) and torch.equal(out.cpu()[inside], y.cpu()[inside])
    if not fp8:
        x = x.clone().requires_grad_()
        w = w.clone().requires_grad_()
        g = torch.full((t, 136), float("nan"), device="cuda", dtype=torch.bfloat16)
        g[21:int(off[-1])] = 1.0
        grouped_matmul(x, w, off).backward(g)
        assert not x.grad.cpu()[~inside].any() and bool(w.grad.isfinite().all())


@pytest.mark.parametrize("n, dtype", [(37, torch.bfloat16), (64, torch.float16), (9, torch.float32), (264, torch.float32)])
def test_long_padding_is_zeroed(n, dtype):
    t, off = 20_000, bounds([3, 0, 70], first=9000)
    x, w = randn(t, 32), B.quantize(randn(3, n, 32, seed=1), rows=128)
    big = torch.full((t * n + 4096,), 3.0, device="cuda", dtype=dtype)      # what the allocator may hand out next
    del big
    y = grouped_matmul(B.quantize(x), w, off, dtype=dtype)
    assert not y[:9000].any() and not y[9073:].any() and bool(y[9000:9073].any())


def test_nan_stays_in_its_group():
    # the last step of a group's contraction reaches rows of the next: they must not count, whatever they hold
    off = bounds([10, 70, 20])
    x, g = randn(100, 64), randn(100, 72, seed=1)
    w = randn(3, 72, 64, seed=2).requires_grad_()
    x[10:80] = float("nan")
    g[10:80] = float("inf")
    grouped_matmul(x, w, off).backward(g)
    assert bool(w.grad[0].isfinite().all() and w.grad[2].isfinite().all() and w.grad[1].isnan().all())
    for i, (lo, hi) in ((0, (0, 10)), (2, (80, 100))):
        O.check_product(w.grad[i], g[lo:hi].t(), x[lo:hi].t())


def test_layouts():
    off, sizes = bounds([50, 20, 90]), (160, 96, 72)
    t, k, n = sizes
    wide, w = randn(t, 2 * k + 3), randn(3, k, n, seed=1)
    views = [wide[:, :k], wide[:, 3:3 + k], wide[:, ::2][:, :k], randn(k, t, seed=4).t()]
    for x in views:
        for weight in (w.transpose(1, 2), w.transpose(1, 2).contiguous(), w[:, :, 1:65].transpose(1, 2), w[:1].expand(3, k, n).transpose(1, 2)):
            y = grouped_matmul(x, weight, off)
            xr, wr = x.contiguous().requires_grad_(), weight.contiguous().requires_grad_()
            xv, wv = x.detach().requires_grad_(), weight.detach().requires_grad_()
            z = grouped_matmul(xr, wr, off)
            assert torch.equal(y, z.detach())
            g = randn(*y.shape, seed=5)
            a, b = torch.autograd.grad(z, (xr, wr), g)
            c, d = torch.autograd.grad(grouped_matmul(xv, wv, off), (xv, wv), g)
            assert torch.equal(a, c) and torch.equal(b, d)
    out = torch.zeros(t, 3 * n, device="cuda", dtype=torch.bfloat16)
    grouped_matmul(views[0], w.transpose(1, 2), off, out=out[:, 5:5 + n])
    assert torch.equal(out[:, 5:5 + n], grouped_matmul(views[0], w.transpose(1, 2), off))
    assert not out[:, :5].any() and not out[:, 5 + n:].any()


def test_bounds_outside_the_rows_are_moved():
    x, w = randn(50, 64), randn(3, 32, 64, seed=1)
    off = torch.tensor([-5, 20, 15, 900], dtype=torch.int32).cuda()     # as [0, 20, 20, 50]
    want = grouped_matmul(x, w, torch.tensor([0, 20, 20, 50], dtype=torch.int32).cuda())
    assert torch.equal(grouped_matmul(x, w, off), want)


def test_many_groups():
    sizes = [i % 3 for i in range(1024)]
    off, x, w = bounds(sizes), randn(sum(sizes), 32), randn(1024, 16, 32, seed=1)
    y = grouped_matmul(x, w, off).double().cpu()
    group = torch.repeat_interleave(torch.arange(1024), torch.tensor(sizes))
    want = torch.einsum("tk,tnk->tn", x.double().cpu(), w.double().cpu()[group])
    terms = torch.einsum("tk,tnk->tn", x.abs().double().cpu(), w.abs().double().cpu()[group])
    O.check(y, want, 33 * 2.0 ** -23 * terms + O.half_step(want.abs() + 33 * 2.0 ** -23 * terms, torch.bfloat16))


def test_empty():
    off = torch.zeros(4, dtype=torch.int32).cuda()
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = randn(3, 32, 64).requires_grad_()
    y = grouped_matmul(x, w, off)
    y.sum().backward()
    assert tuple(y.shape) == (0, 32) and tuple(x.grad.shape) == (0, 64) and not w.grad.any()
    x = randn(9, 64).requires_grad_()       # rows, but no group has any
    w.grad = None
    y = grouped_matmul(x, w, off)
    y.sum().backward()
    assert not y.any() and not x.grad.any() and not w.grad.any()


def test_graph_replays_with_other_bounds():
    x, w, off = randn(90, 64), randn(4, 48, 64, seed=1), bounds([40, 0, 20, 30])
    kept = B.quantize(w, rows=128)
    wt = w.clone().requires_grad_()

    def step():
        y = grouped_matmul(x, wt, off)
        return y, grouped_matmul(x, kept, off), *torch.autograd.grad(y.float().square().sum(), wt)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for sizes in ([0, 0, 90, 0], [1, 2, 3, 4], [40, 0, 20, 30]):
        off.copy_(bounds(sizes))
        graph.replay()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("sizes", [[2048] * 8, [512] * 32, [0, 4992, 512, 1472, 9408], [4992, 517, 1472, 9403]], ids=str)
def test_weight_gradient_of_long_groups(sizes):
    # hundreds of steps without a partial one, and between partial ones
    t, off = sum(sizes), bounds(sizes)
    x, g = randn(t, 1024), randn(t, 512, seed=1)
    w = torch.zeros(len(sizes), 512, 1024, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    first = None
    for _ in range(10):
        (dw,) = torch.autograd.grad(grouped_matmul(x, w, off), w, g)
        first = dw if first is None else first
        assert torch.equal(dw, first)
    for i, (lo, hi) in enumerate(spans(off)):
        a, b = g[lo:hi].double().t(), x[lo:hi].double()
        terms, want = (a.abs() @ b.abs()).cpu(), (a @ b).cpu()
        acc = (hi - lo + 1) * 2.0 ** -23 * terms
        O.check(first[i], want, acc + O.half_step(want.abs() + acc, torch.bfloat16))


@pytest.mark.parametrize("k, n", [(2048, 1024), (2304, 2200), (8192, 96), (520, 2048)])
@pytest.mark.parametrize("sizes", [[1500, 5, 0, 300, 64, 1], [3, 2, 900, 1, 0, 0, 40, 2, 800, 7], [256] * 6], ids=str)
def test_weight_gradient_of_unequal_groups(sizes, k, n):
    # more tiles than CTAs and one group far above the mean: tiles are dealt out, every one once
    t, off = sum(sizes), bounds(sizes)
    x, g = randn(t, k), randn(t, n, seed=1)
    w = torch.zeros(len(sizes), n, k, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    (dw,) = torch.autograd.grad(grouped_matmul(x, w, off), w, g)
    for i, (lo, hi) in enumerate(spans(off)):
        a, b = g[lo:hi].double().t(), x[lo:hi].double()
        terms, want = a.abs() @ b.abs(), a @ b
        acc = (hi - lo + 1) * 2.0 ** -23 * terms
        half = torch.maximum((want.abs() + acc) * 2.0 ** -8, torch.full_like(want, 1e-38))
        assert bool(((dw[i].double() - want).abs() <= acc + half).all())


def test_first_call_in_a_new_thread():
    # a thread without a CUDA context of its own, as autograd's
    from concurrent.futures import ThreadPoolExecutor
    x, w, off = randn(8, 64), randn(2, 32, 64), bounds([3, 5])
    with ThreadPoolExecutor(1) as pool:
        y = pool.submit(grouped_matmul, x, w, off).result()
    torch.cuda.synchronize()
    assert torch.equal(y, grouped_matmul(x, w, off))


def test_output_of_more_than_two_to_the_31_elements():
    t, n, k = 140_000, 16384, 64
    off = torch.tensor([0, 70_001, t], dtype=torch.int32).cuda()
    x, w = randn(t, k), randn(2, n, k, seed=1)
    y = grouped_matmul(x, w, off)
    for lo, hi, e in ((0, 50, 0), (69_980, 70_001, 0), (70_001, 70_030, 1), (t - 50, t, 1)):
        O.check_product(y[lo:hi], x[lo:hi], w[e])


def test_refusals_on_the_gpu():
    x, w, off = randn(8, 64), randn(2, 32, 64), bounds([3, 5])
    with pytest.raises(ValueError, match="without gradients"):
        grouped_matmul(x.clone().requires_grad_(), B.quantize(w, rows=128), off)
    with pytest.raises(ValueError, match="without gradients"):
        grouped_matmul(x.clone().requires_grad_(), w, off, out=torch.empty(8, 32, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="CUDA tensors"):
        grouped_matmul(x, w, off.cpu())
