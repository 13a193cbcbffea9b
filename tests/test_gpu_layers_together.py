"""The block-scaled FP8 layer, the grouped products and the training reconstruction in one training
step, as a controller with expert layers would run them: pixels routed to experts, a 1x1 layer 64 -> 64 on
the metadata grid, reconstruct, loss, backward.  Each gradient is checked against the plain 64-bit form at the
tensors that this very step produced."""
import numpy as np
import pytest
import torch

import block_oracle as O
from aeisu_b200 import block_fp8 as B
from aeisu_b200.grouped import grouped_matmul
from aeisu_b200.reconstruction import reconstruct
from oracle import reconstruct_np as R
from test_gpu_reconstruct import inputs
from test_reconstruct_oracle import rel

pytestmark = pytest.mark.gpu


def routed(pixels, experts, gen):
    """Rows sorted by expert: (order, offsets)."""
    e = torch.randint(0, experts - 1, (pixels,), generator=gen)     # the last expert has none
    order = torch.argsort(e, stable=True)
    return order.cuda(), torch.cat([torch.zeros(1, dtype=torch.int64), torch.bincount(e, minlength=experts).cumsum(0)]
                                   ).to(torch.int32).cuda()


def test_training_step_through_experts_linear_and_reconstruct():
    b, h, w, experts = 2, 36, 44, 4
    src, _, base, basis, grad = inputs(17, b, h, w, 4)
    gen = torch.Generator().manual_seed(3)
    rows = b * (h // 2) * (w // 2)
    features = torch.randn(rows, 64, generator=gen).bfloat16().cuda()
    order, off = routed(rows, experts, gen)
    we = (torch.randn(experts, 64, 64, generator=gen) / 8).bfloat16().cuda().requires_grad_()
    wt = (torch.randn(64, 64, generator=gen) / 8).cuda().requires_grad_()          # float32 master weight
    bt = torch.randn(64, generator=gen).cuda().requires_grad_()
    base_t, basis_t = (torch.from_numpy(v).cuda().requires_grad_() for v in (base, basis))

    x = features[order].requires_grad_()
    hidden = grouped_matmul(x, we, off)
    hidden.retain_grad()
    back = torch.empty_like(order)
    back[order] = torch.arange(rows, device="cuda")
    act = torch.nn.functional.leaky_relu(hidden[back], 0.1)
    act.retain_grad()
    out = B.linear(act.reshape(b, h // 2, w // 2, 64), wt, bt)
    out.retain_grad()
    meta = out.permute(0, 3, 1, 2)
    hr = reconstruct(torch.from_numpy(src).cuda(), meta, base_t, basis_t, trim=4)
    hr.backward(torch.from_numpy(grad).cuda())
    torch.cuda.synchronize()

    a, g = act.detach(), out.grad.reshape(rows, 64)
    assert out.dtype == torch.bfloat16 and g.dtype == torch.bfloat16
    O.check_product(out.detach().reshape(rows, 64), O.values(a), O.values(wt.detach(), 128), bt.detach())
    m32 = meta.detach().float().cpu().numpy()
    want_m, want_b, want_k = R.reconstruct_backward(src, m32, base, basis, grad, 4, 1, 0)
    assert rel(hr.detach().cpu().numpy(), R.reconstruct(src, m32, base, basis, 4)) < 2e-6
    assert rel(base_t.grad.cpu().numpy(), want_b) < 2e-5 and rel(basis_t.grad.cpu().numpy(), want_k) < 2e-5
    # the metadata gradient, rounded to bfloat16: half a step of it and the reconstruction's own 2e-6 of the largest
    got = out.grad.permute(0, 3, 1, 2).float().cpu().numpy()
    assert np.all(np.abs(got - want_m) <= np.abs(want_m) * 2.0 ** -8 + 2.1e-6 * np.abs(want_m).max())
    O.check_product(act.grad, O.values(g), O.values(wt.detach().t(), 128))
    O.check_product(wt.grad, O.values(g.t()), O.values(a.t()))
    s = g.double().cpu()
    O.check(bt.grad, s.sum(0), (rows + 1) * 2.0 ** -24 * s.abs().sum(0))
    gh = hidden.grad
    for i, (lo, hi) in enumerate(zip(off.tolist(), off.tolist()[1:])):
        O.check_product(hidden[lo:hi], x.detach()[lo:hi], we.detach()[i])
        O.check_product(x.grad[lo:hi], gh[lo:hi], we.detach()[i].t())
        O.check_product(we.grad[i], gh[lo:hi].t(), x.detach()[lo:hi].t())
    assert not we.grad[-1].any()


def test_serving_keeps_weights_in_fp8():
    # the same layers served: weights quantised once, a frame's pixels through experts and layer, one graph
    gen = torch.Generator().manual_seed(4)
    rows, experts = 1000, 4
    x = torch.randn(rows, 64, generator=gen).bfloat16().cuda()
    order, off = routed(rows, experts, gen)
    x = x[order]
    we = B.quantize((torch.randn(experts, 64, 64, generator=gen) / 8).cuda(), rows=128)
    wt = B.quantize((torch.randn(64, 64, generator=gen) / 8).cuda(), rows=128)
    bt = torch.randn(64, generator=gen).bfloat16().cuda()

    def step():
        h = grouped_matmul(x, we, off)
        return h, B.linear(h, wt, bt)

    h, y = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        graph.replay()
    assert torch.equal(captured[0], h) and torch.equal(captured[1], y)
    xv, wv = O.values(x), we.dequantize()
    for i, (lo, hi) in enumerate(zip(off.tolist(), off.tolist()[1:])):
        O.check_product(h[lo:hi], xv[lo:hi], wv[i])
    O.check_product(y, O.values(h), wt.dequantize(), bt)
