"""Measured cases of the block-scaled FP8 operators and the products grouped by expert.

Three operators: ``quantize`` (to 8-bit floating point with one power-of-two scale for each block
of 128), ``linear`` / ``matmul`` on such operands, and ``grouped_matmul`` (rows sorted by expert,
ragged group sizes).  With ``own`` false ``run`` computes them from elementary torch operations in
32 bits; with ``own`` true it calls ``aeisu_b200.block_fp8`` and ``aeisu_b200.grouped``.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_CODES = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
# the largest finite code is 0.875 * 2**_TOP
_TOP = {torch.float8_e4m3fn: 9, torch.float8_e5m2: 16}


def listed():
    return [
        # one token's activations on their way into an FP8 layer: latency alone
        {"name": "quantize-token", "op": "quantize", "m": 1, "k": 4096, "rows": 1, "both": False, "dtype": "bf16",
         "codes": "e4m3"},
        # the activations of a training step, in both directions: rows for the product, columns for the
        # weight gradient
        {"name": "quantize-train", "op": "quantize", "m": 8192, "k": 4096, "rows": 1, "both": True, "dtype": "bf16",
         "codes": "e4m3"},
        # an FP32 master weight of odd size to 128 x 128 blocks, in both directions
        {"name": "quantize-weight-odd", "op": "quantize", "m": 2049, "k": 5003, "rows": 128, "both": True,
         "dtype": "fp32", "codes": "e5m2"},
        # a layer answering one token, weights kept in FP8
        {"name": "linear-token", "op": "linear", "m": 1, "k": 4096, "n": 4096, "bias": False, "dtype": "bf16"},
        # a small ragged batch through a layer of odd size with a bias
        {"name": "linear-rows-odd", "op": "linear", "m": 37, "k": 2000, "n": 1001, "bias": True, "dtype": "fp16"},
        # training the controller's 1x1 layer 128 -> 64 on 32 sources of 288 x 288 (a 72 x 72 grid each)
        {"name": "train-controller", "op": "train", "m": 165888, "k": 128, "n": 64, "bias": True, "dtype": "bf16"},
        # a training step of an ordinary wide layer
        {"name": "train-wide", "op": "train", "m": 8192, "k": 4096, "n": 4096, "bias": False, "dtype": "bf16"},
        # the largest: a long batch through a wide layer, both operands in FP8 already
        {"name": "matmul-large", "op": "matmul", "m": 16384, "k": 8192, "n": 8192, "dtype": "bf16"},
        # experts answering a few tokens, weights kept in FP8; most experts have no row
        {"name": "experts-decode", "op": "experts", "t": 16, "e": 32, "k": 2048, "n": 1024, "dtype": "bf16",
         "skew": 1.0},
        # experts over a long batch, weights kept in FP8
        {"name": "experts-prefill", "op": "experts", "t": 8192, "e": 64, "k": 2048, "n": 2048, "dtype": "bf16",
         "skew": 0.5},
        # training the experts of a layer, groups of very unequal size
        {"name": "experts-train", "op": "experts_train", "t": 16384, "e": 16, "k": 2048, "n": 1024, "dtype": "bf16",
         "skew": 1.0},
        # the same with odd sizes
        {"name": "experts-train-odd", "op": "experts_train", "t": 1003, "e": 5, "k": 200, "n": 76, "dtype": "fp16",
         "skew": 1.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo, hi):
    """A layer's width: mostly a multiple of 16, now and then any number."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.3 else max(lo, n // 16 * 16)


def draw(rng):
    op = rng.choice(["quantize", "linear", "train", "matmul", "experts", "experts_train"])
    half = rng.choice(["bf16", "fp16"])
    if op == "quantize":
        return {"op": op, "m": _log(rng, 1, 8192), "k": _width(rng, 16, 6000), "rows": rng.choice([1, 128]),
                "both": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "codes": rng.choice(["e4m3", "e5m2"])}
    if op == "linear":
        return {"op": op, "m": _log(rng, 1, 500), "k": _width(rng, 32, 8192), "n": _width(rng, 16, 8192),
                "bias": rng.random() < 0.5, "dtype": half}
    if op == "train":
        return {"op": op, "m": _log(rng, 100, 16384), "k": _width(rng, 32, 4096), "n": _width(rng, 32, 4096),
                "bias": rng.random() < 0.5, "dtype": half}
    if op == "matmul":
        return {"op": op, "m": _log(rng, 1, 16384), "k": _width(rng, 64, 8192), "n": _width(rng, 64, 8192), "dtype": half}
    if op == "experts":
        return {"op": op, "t": _log(rng, 1, 8192), "e": _log(rng, 2, 64), "k": _width(rng, 64, 2048),
                "n": _width(rng, 64, 2048), "dtype": half, "skew": rng.choice([0.0, 0.5, 1.0, 2.0])}
    return {"op": op, "t": _log(rng, 100, 16384), "e": _log(rng, 2, 32), "k": _width(rng, 32, 2048),
            "n": _width(rng, 32, 1024), "dtype": half, "skew": rng.choice([0.0, 0.5, 1.0])}


# ---- inputs ----------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, scale, dtype):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _activations(g, shape, dtype):
    """Normal values; a few columns carry outliers, and one value in a thousand is zero."""
    x = torch.randn(shape, generator=g, device="cuda")
    x *= 1.0 + 15.0 * (torch.rand(shape[-1], generator=g, device="cuda") < 0.01)
    x *= torch.rand(shape, generator=g, device="cuda") >= 0.001
    return x.to(dtype)


def _offsets(g, t, e, skew):
    """Row bounds of e groups that hold all t rows, sizes by a random popularity exp(skew * normal);
    one expert is never chosen."""
    share = torch.exp(skew * torch.randn(e, generator=g, device="cuda"))
    share[e // 2] = 0.0
    chosen = torch.multinomial(share, t, replacement=True, generator=g)
    sizes = torch.bincount(chosen, minlength=e)
    return torch.cat([sizes.new_zeros(1), sizes.cumsum(0)]).to(torch.int32), int(sizes.max())


def prepare(case, seed):
    g = _generator(seed)
    op, dt = case["op"], _DTYPES[case["dtype"]]
    s = {"case": case}
    if op == "quantize":
        s["x"] = _activations(g, (case["m"], case["k"]), dt)
    elif op in ("linear", "train", "matmul"):
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = _activations(g, (m, k), dt)
        s["w"] = _randn(g, (n, k), k ** -0.5, dt)
        s["b"] = _randn(g, (n,), 0.1, dt) if case.get("bias") else None
        if op == "linear":      # the weights are kept in FP8
            s["wq"] = _quantize(s.pop("w"), 128, torch.float8_e4m3fn)
        elif op == "matmul":    # both operands are
            s["xq"] = _quantize(s.pop("x"), 1, torch.float8_e4m3fn)
            s["wq"] = _quantize(s.pop("w"), 128, torch.float8_e4m3fn)
        else:
            s["g"] = _randn(g, (m, n), 1e-3, dt)
    else:
        t, e, k, n = case["t"], case["e"], case["k"], case["n"]
        s["x"] = _activations(g, (t, k), dt)
        s["w"] = _randn(g, (e, n, k), k ** -0.5, dt)
        s["off"], s["cap"] = _offsets(g, t, e, case["skew"])
        if op == "experts":
            s["wq"] = _quantize(s.pop("w"), 128, torch.float8_e4m3fn)
        else:
            s["g"] = _randn(g, (t, n), 1e-3, dt)
    for name in ("x", "w", "b"):
        if op in ("train", "experts_train") and s.get(name) is not None:
            s[name].requires_grad_()
    return s


# ---- the plain form --------------------------------------------------------------------------


def _quantize(x, rows, codes):
    """(codes, scales) of x [..., R, C]: scales [..., ceil(C / 128), ceil(R / rows)] as E8M0."""
    r, c = x.shape[-2:]
    rb, cb = -(-r // rows), -(-c // 128)
    f = torch.nn.functional.pad(x.float(), (0, cb * 128 - c, 0, rb * rows - r))
    f = f.reshape(*x.shape[:-2], rb, rows, cb, 128)
    amax = torch.where(f.isfinite(), f.abs(), 0.0).amax((-3, -1), keepdim=True)
    m, e = torch.frexp(amax)                                  # amax = m * 2**e, 0.5 <= m < 1
    e = torch.where(amax > 0, e - _TOP[codes] + (m > 0.875), 0).clamp(-127, 127)
    q = torch.where(f.isfinite(), f, math.nan) * torch.ldexp(torch.ones_like(amax), -e)
    q = q.reshape(*x.shape[:-2], rb * rows, cb * 128)[..., :r, :c].to(codes)
    scales = (e + 127).to(torch.uint8).reshape(*x.shape[:-2], rb, cb).transpose(-1, -2).contiguous()
    return q.contiguous(), scales.view(torch.float8_e8m0fnu)


def _values(q, rows, real=torch.float32):
    """What a block-scaled operand stands for."""
    codes, scales = q
    r, c = codes.shape[-2:]
    s = scales.to(real).transpose(-1, -2).repeat_interleave(rows, -2)[..., :r, :]
    return codes.to(real) * s.repeat_interleave(128, -1)[..., :c]


def _padded_groups(off, cap, t):
    """Row index of place i of each group [e, cap] (t where the group is shorter)."""
    at = off[:-1, None].long() + torch.arange(cap, device=off.device)
    return torch.where(at < off[1:, None], at, t)


def _gather(x, at):
    return torch.cat([x.float(), x.new_zeros(1, x.shape[1]).float()])[at]


def _scatter(y, at, t):
    out = y.new_zeros(t + 1, y.shape[-1])
    out[at.reshape(-1)] = y.reshape(-1, y.shape[-1])
    return out[:t]


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    e4 = torch.float8_e4m3fn
    if op == "quantize":
        out = [_quantize(s["x"], case["rows"], _CODES[case["codes"]])]
        if case["both"]:
            out.append(_quantize(s["x"].t(), case["rows"], _CODES[case["codes"]]))
        return out
    if op == "matmul":
        return (_values(s["xq"], 1) @ _values(s["wq"], 128).t()).to(_DTYPES[case["dtype"]])
    if op == "experts":
        t, dt = case["t"], s["x"].dtype
        at = _padded_groups(s["off"], s["cap"], t)
        x = _values(_quantize(s["x"], 1, e4), 1)
        y = torch.bmm(_gather(x, at), _values(s["wq"], 128).transpose(1, 2))
        return _scatter(y, at, t).to(dt)
    with torch.no_grad():
        if op == "experts_train":
            t, dt = case["t"], s["x"].dtype
            at = _padded_groups(s["off"], s["cap"], t)
            x, g, w = _gather(s["x"], at), _gather(s["g"], at), s["w"].float()
            y = _scatter(torch.bmm(x, w.transpose(1, 2)), at, t)
            dx = _scatter(torch.bmm(g, w), at, t)
            return {"y": y.to(dt), "dx": dx.to(dt), "dw": torch.bmm(g.transpose(1, 2), x).to(dt)}
        x, dt = s["x"], s["x"].dtype
        wq = s["wq"] if op == "linear" else _quantize(s["w"], 128, e4)
        y = _values(_quantize(x, 1, e4), 1) @ _values(wq, 128).t()
        if s["b"] is not None:
            y = y + s["b"].float()
        if op == "linear":
            return y.to(dt)
        g = s["g"]
        dx = _values(_quantize(g, 1, e4), 1) @ _values(wq, 128)
        dw = _values(_quantize(g.t(), 1, e4), 1) @ _values(_quantize(x.t(), 1, e4), 1).t()
        out = {"y": y.to(dt), "dx": dx.to(dt), "dw": dw.to(dt)}
        if s["b"] is not None:
            out["db"] = g.float().sum(0).to(dt)
        return out


# ---- the framework's calls -------------------------------------------------------------------


def _framework(s):
    from aeisu_b200 import block_fp8, grouped
    case, op = s["case"], s["case"]["op"]
    if op == "quantize":
        codes = _CODES[case["codes"]]
        if case["both"]:
            q, qt = block_fp8.quantize_both(s["x"], rows=case["rows"], dtype=codes)
            return [(q.codes, q.scales), (qt.codes, qt.scales)]
        q = block_fp8.quantize(s["x"], rows=case["rows"], dtype=codes)
        return [(q.codes, q.scales)]
    if op == "matmul":
        return block_fp8.matmul(block_fp8.BlockFP8(*s["xq"], rows=1), block_fp8.BlockFP8(*s["wq"], rows=128),
                                dtype=_DTYPES[case["dtype"]])
    if op == "linear":
        return block_fp8.linear(s["x"], block_fp8.BlockFP8(*s["wq"], rows=128), s["b"])
    if op == "experts":
        return grouped.grouped_matmul(s["x"], block_fp8.BlockFP8(*s["wq"], rows=128), s["off"])
    if op == "experts_train":
        y = grouped.grouped_matmul(s["x"], s["w"], s["off"])
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["g"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    y = block_fp8.linear(s["x"], s["w"], s["b"])
    leaves = (s["x"], s["w"]) + (() if s["b"] is None else (s["b"],))
    grads = torch.autograd.grad(y, leaves, s["g"])
    return {"y": y.detach(), **dict(zip(("dx", "dw", "db"), grads))}


def run(state):
    return _framework(state) if own else _plain(state)


# ---- what a pass cannot do without -----------------------------------------------------------


def work(case):
    op, b = case["op"], _BYTES[case["dtype"]]
    if op == "quantize":
        values = case["m"] * case["k"]
        ways = 2 if case["both"] else 1
        return {"bytes": values * b + ways * (values + values / (128 * case["rows"])), "flops": 2 * values * ways}
    k, n = case["k"], case["n"]
    if op == "linear":
        m = case["m"]
        return {"bytes": m * k * b + n * k * (1 + 1 / 16384) + m * n * b + (n * b if case["bias"] else 0),
                "flops": 2 * m * n * k}
    if op == "matmul":
        m = case["m"]
        return {"bytes": m * k * (1 + 1 / 128) + n * k * (1 + 1 / 16384) + m * n * b, "flops": 2 * m * n * k}
    if op == "train":
        m = case["m"]
        return {"bytes": b * (2 * m * k + 2 * n * k + 2 * m * n + (2 * n if case["bias"] else 0)),
                "flops": 6 * m * n * k}
    t, e = case["t"], case["e"]
    if op == "experts":
        # an expert without a row is not read; how many have one depends on the seed, at most t
        return {"bytes": t * k * b + min(e, t) * n * k * (1 + 1 / 16384) + t * n * b, "flops": 2 * t * n * k}
    return {"bytes": b * (2 * t * k + 2 * e * n * k + 2 * t * n), "flops": 6 * t * n * k}


# ---- the definition, in 64 bits --------------------------------------------------------------


def _blocks64(x, rows, codes):
    """(values of the codes, scales) of a matrix, by the definition: the smallest power of two s with
    amax / s no larger than the largest code, then the nearest code (ties to even)."""
    bits, least, most = (3, -6, 448.0) if codes == "e4m3" else (2, -14, 57344.0)
    x = x.detach().double()
    r, c = x.shape
    tall = torch.arange(r, device=x.device) // rows
    wide = torch.arange(c, device=x.device) // 128
    cell = tall[:, None] * (int(wide[-1]) + 1) + wide
    amax = torch.zeros(int(cell[-1, -1]) + 1, dtype=torch.float64, device=x.device)
    amax.scatter_reduce_(0, cell.reshape(-1), x.abs().reshape(-1), "amax")
    p = torch.ceil(torch.log2(amax / most))
    p = p - (torch.exp2(p - 1) * most >= amax).double()      # the logarithm may be off by a step
    p = p + (torch.exp2(p) * most < amax).double()
    scale = torch.exp2(torch.where(amax > 0, p, 0.0).clamp(-127, 127))
    v = x / scale[cell]
    _, e = torch.frexp(v)
    step = torch.exp2(torch.maximum(e.double() - 1, torch.tensor(float(least), device=x.device)) - bits)
    return torch.round(v / step) * step, scale, cell


def _stand64(x, rows):
    v, scale, cell = _blocks64(x, rows, "e4m3")
    return v * scale[cell]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        out = []
        for x in (s["x"], s["x"].t())[:2 if case["both"] else 1]:
            v, scale, _ = _blocks64(x, case["rows"], case["codes"])
            out.append((v, scale.reshape(-1, -(-x.shape[1] // 128)).t().contiguous()))
        return out
    if op == "matmul":
        return _values(s["xq"], 1, torch.float64) @ _values(s["wq"], 128, torch.float64).t()
    if op == "linear":
        y = _stand64(s["x"], 1) @ _values(s["wq"], 128, torch.float64).t()
        return y if s["b"] is None else y + s["b"].double()
    if op == "train":
        x, w, g = s["x"].detach(), _stand64(s["w"], 128), s["g"]
        y = _stand64(x, 1) @ w.t()
        out = {"y": y if s["b"] is None else y + s["b"].detach().double(), "dx": _stand64(g, 1) @ w,
               "dw": _stand64(g.t(), 1) @ _stand64(x.t(), 1).t()}
        if s["b"] is not None:
            out["db"] = g.double().sum(0)
        return out
    off = s["off"].tolist()
    spans = [slice(a, b) for a, b in zip(off, off[1:])]
    if op == "experts":
        x, w = _stand64(s["x"], 1), _values(s["wq"], 128, torch.float64)
        return torch.cat([x[p] @ w[i].t() for i, p in enumerate(spans)])
    x, w, g = s["x"].detach().double(), s["w"].detach().double(), s["g"].double()
    return {"y": torch.cat([x[p] @ w[i].t() for i, p in enumerate(spans)]),
            "dx": torch.cat([g[p] @ w[i] for i, p in enumerate(spans)]),
            "dw": torch.stack([g[p].t() @ x[p] for p in spans])}
