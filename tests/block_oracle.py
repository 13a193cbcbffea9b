"""Plain 64-bit forms of the block-scaled FP8 operators and the grouped products, and the error
bounds that the tests use.

A product accumulates K terms in float32.  Whatever the order, and even if every addition
truncates, the result is off by at most ``K * 2**-23`` times the sum of the terms' magnitudes; the
final rounding adds half a step of the output's type, relative to the value (or half the smallest
subnormal).
"""
import torch

TOP = {torch.float8_e4m3fn: (448.0, 3, -6), torch.float8_e5m2: (57344.0, 2, -14)}   # largest, mantissa bits, least exponent


def quantize(x, rows, dtype):
    """(code values float64, scales float64 [RB, CB]) of a matrix, block by block, by the definition."""
    x = x.double().cpu()
    top, bits, least = TOP[dtype]
    r, c = x.shape
    rb, cb = -(-r // rows), -(-c // 128)
    v, s = torch.empty_like(x), torch.empty(rb, cb, dtype=torch.float64)
    for i in range(rb):
        for j in range(cb):
            b = x[i * rows:(i + 1) * rows, j * 128:(j + 1) * 128]
            fine = b.isfinite()
            amax = float(torch.where(fine, b.abs(), 0.0).max())
            e = 0
            if amax > 0:
                e = -127
                while amax / 2.0 ** e > top:
                    e += 1
            q = torch.where(fine, b, float("nan")) / 2.0 ** e
            step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** least))) - bits)
            s[i, j] = 2.0 ** e
            v[i * rows:(i + 1) * rows, j * 128:(j + 1) * 128] = torch.round(q / step) * step
    return v, s


def values(x, rows=1, dtype=torch.float8_e4m3fn):
    """What the quantised matrix stands for."""
    v, s = quantize(x, rows, dtype)
    r, c = x.shape
    return v * s.repeat_interleave(rows, 0)[:r].repeat_interleave(128, 1)[:, :c]


def half_step(y, dtype):
    """Half a rounding step of `dtype` at y."""
    f = torch.finfo(dtype)
    return torch.maximum(y.abs() * (f.eps / 2), torch.tensor(f.smallest_normal * f.eps / 2, dtype=torch.float64))


def product_bound(a, b, dtype, y, extra=0):
    """Largest error of y = a @ b.T held in float32 and rounded to `dtype`."""
    terms = a.abs() @ b.abs().t()
    acc = (a.shape[1] + 1 + extra) * 2.0 ** -23 * terms
    return acc + half_step(y.abs() + acc, dtype)


def check_product(got, a, b, bias=None):
    """got against a @ b.T + bias of float64 matrices, within the bound, NaN where it is NaN."""
    a, b = a.double().cpu(), b.double().cpu()
    y = a @ b.t()
    bound = product_bound(a, b, got.dtype, y)
    if bias is not None:
        add = bias.double().cpu()
        bound = bound + half_step(y + add, got.dtype) + 2.0 ** -23 * add.abs()
        y = y + add
    check(got, y, bound)


def check(got, want, bound):
    # A value rounds to infinity from half a step above the type's largest on (float16: 65504 + 16):
    # one that lies there for certain has to, one that may lie there within the bound may.
    f = torch.finfo(got.dtype)
    over = f.max * (1 + f.eps / 4)
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan())
    bound = bound.expand_as(want)
    may, must = want.abs() + bound >= over, want.abs() - bound >= over
    inf = got.isinf() & (got.sign() == want.sign())
    assert bool(inf[must].all())
    fine = ~want.isnan() & ~(may & inf)
    err = (got - want).abs()[fine]
    assert bool((err <= bound.expand_as(want)[fine]).all()), f"off by up to {float((err / bound.expand_as(want)[fine]).max()):.3g} bounds"
