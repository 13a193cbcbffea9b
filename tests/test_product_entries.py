"""The C entry points of block-scaled FP8 and grouped products, without a GPU: every argument that a
kernel or the host arithmetic could not stand is refused before any of it runs."""
import pytest
import torch
from torch.autograd import forward_ad

from aeisu_b200 import _lib, block_fp8 as B, build
from aeisu_b200.grouped import grouped_matmul
from test_block_fp8 import HALF, blocks, packed


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def refused(call, text):
    assert call() == _lib.INVALID_ARG and text in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize("empty", [dict(rows=0), dict(cols=0), dict(batch=0), dict(rows=-5), dict(batch=-1)], ids=str)
def test_entries_refuse_empty_matrices(lib, empty):
    # (a division by the number of groups, or by that of row tiles, ended the process)
    codes, half, out = packed(), packed(**HALF), packed(cols=8, ld=8, **HALF)
    bad, few = packed(**empty), packed(**{**HALF, **empty})
    none = packed(**{**HALF, "cols": 8, "ld": 8, **empty})
    ws = (4096, 1 << 20, 0, None)
    for call in (lambda: lib.aeisu_linear(half, bad, None, 0, out, *ws),
                 lambda: lib.aeisu_linear(few, codes, None, 0, none, *ws),
                 lambda: lib.aeisu_linear_forward(half, few, None, 0, out, None, None, *ws),
                 lambda: lib.aeisu_linear_backward(few, 8, 3, None, None, None, 2, None, 2, None, 2, *ws),
                 lambda: lib.aeisu_grouped_linear(half, bad, 4096, 1, out, *ws),
                 lambda: lib.aeisu_grouped_linear(few, codes, 4096, 1, none, *ws),
                 lambda: lib.aeisu_grouped_product(half, few, 4096, 1, out, 0, None),
                 lambda: lib.aeisu_grouped_weight_gradient(half, few, 4096, 2, 4096, 2, 0, None),
                 lambda: lib.aeisu_column_sum(few, 4096, 2, 4096, 1 << 20, 0, None),
                 lambda: lib.aeisu_block_quantize(few, 1, bad, None, 0, None),
                 lambda: lib.aeisu_product(bad, codes, None, 0, none, None, 0, 0, None)):
        refused(call, "sizes are out of range")


@pytest.mark.parametrize("place, bad, text", [
    ("grad_x", "pointer", "output"), ("grad_weight", "pointer", "output"), ("grad_bias", "pointer", "output"),
    ("grad_x", "type", "output"), ("grad_weight", "type", "output"), ("grad_bias", "type", "output"),
    ("kept_x", "pointer", "kept"), ("kept_weight", "pointer", "kept")])
def test_linear_backward_refuses_what_it_cannot_store(lib, place, bad, text):
    args = dict(kept_x=4096, kept_weight=4096, grad_x=4096, grad_weight=4096, grad_bias=4096)
    types = dict(grad_x=0, grad_weight=0, grad_bias=0)
    if bad == "type":
        types[place] = 3
    else:
        args[place] += 2
    refused(lambda: lib.aeisu_linear_backward(
        packed(**HALF), 64, 3, args["kept_x"], args["kept_weight"], args["grad_x"], types["grad_x"], args["grad_weight"],
        types["grad_weight"], args["grad_bias"], types["grad_bias"], 4096, 1 << 30, 0, None), text)


def test_other_entries_refuse_what_they_cannot_store(lib):
    codes, half, out = packed(), packed(**HALF), packed(cols=8, ld=8, **HALF)
    ws = (4096, 1 << 30, 0, None)
    fp8_out, narrow = packed(cols=8, ld=8), packed(cols=8, ld=7, **HALF)
    for call, text in (
            (lambda: lib.aeisu_column_sum(half, 4098, 0, *ws), "output"),
            (lambda: lib.aeisu_column_sum(half, 4097, 2, *ws), "output"),
            (lambda: lib.aeisu_column_sum(half, 4096, 3, *ws), "output"),
            (lambda: lib.aeisu_column_sum(half, 4096, -1, *ws), "output"),
            (lambda: lib.aeisu_column_sum(half, 4096, 2, 4098, 1 << 30, 0, None), "workspace"),
            (lambda: lib.aeisu_product(codes, codes, None, 0, out, 4098, 1 << 30, 0, None), "workspace"),
            (lambda: lib.aeisu_linear_forward(half, half, None, 0, out, 4104, None, *ws), "kept"),
            (lambda: lib.aeisu_linear_forward(half, half, None, 0, out, None, 4104, *ws), "kept"),
            (lambda: lib.aeisu_linear(half, codes, None, 0, fp8_out, *ws), "output"),
            (lambda: lib.aeisu_linear(half, codes, None, 0, narrow, *ws), "output"),
            (lambda: lib.aeisu_linear_forward(half, half, None, 0, fp8_out, None, None, *ws), "output"),
            (lambda: lib.aeisu_grouped_linear(half, codes, 4096, 1, fp8_out, *ws), "output"),
            (lambda: lib.aeisu_grouped_linear(half, codes, 4096, 1, narrow, *ws), "output")):
        refused(call, text)


@pytest.mark.parametrize("which", ["x", "weight", "bias"])
def test_linear_refuses_forward_mode_inputs(which):
    t = dict(x=torch.randn(4, 64), weight=torch.randn(8, 64), bias=torch.randn(8))
    with forward_ad.dual_level():
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        for weight in (t["weight"], t["weight"].clone().requires_grad_(), blocks(8, 64, 128)):
            if which == "weight" and weight is not t["weight"]:
                continue
            with pytest.raises(ValueError, match="forward-mode"):
                B.linear(t["x"], weight, t["bias"])
        with pytest.raises(ValueError, match="CUDA tensors"):     # no dual among them
            B.linear(torch.randn(4, 64), torch.randn(8, 64))


@pytest.mark.parametrize("which", ["x", "weight", "out"])
def test_grouped_products_refuse_forward_mode_inputs(which):
    t = dict(x=torch.randn(6, 16).half(), weight=torch.randn(2, 8, 16).half())
    off = torch.tensor([0, 2, 6], dtype=torch.int32)
    if which == "out":
        t["out"] = torch.zeros(6, 8).half()
    with forward_ad.dual_level():
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(ValueError, match="forward-mode"):
            grouped_matmul(t["x"], t["weight"], off, out=t.get("out"))
        if which == "x":
            with pytest.raises(ValueError, match="forward-mode"):
                grouped_matmul(t["x"], blocks(8, 16, 128, lead=(2,)), off)
    if which != "out":
        with pytest.raises(ValueError, match="forward-mode"):
            torch.func.jvp(lambda v: grouped_matmul(*(v if n == which else t[n] for n in ("x", "weight")), off),
                           (t[which].detach().clone(),), (torch.ones_like(t[which]),))


def test_check_products_raises_what_the_library_reports(monkeypatch):
    seen = []

    class Library:
        code = 1

        def aeisu_product_status(self, index, code):
            seen.append(index)
            code._obj.value, self.code = self.code, 0
            return _lib.OK

    fake = Library()
    monkeypatch.setattr(B, "_call", lambda: fake)
    with pytest.raises(TimeoutError, match="device 2"):
        B.check_products(2)
    for device in (2, "cuda:3", torch.device("cuda", 4)):
        B.check_products(device)
    assert seen == [2, 2, 3, 4]
    with pytest.raises(ValueError, match="CUDA device"):
        B.check_products("cpu")


def test_a_subclass_of_block_fp8_serves_everywhere():
    class Named(B.BlockFP8):
        pass

    def named(q):
        return Named(q.codes, q.scales, q.rows)

    w, experts = named(blocks(8, 64, 128)), named(blocks(8, 64, 128, lead=(2,)))
    x, off = torch.zeros(6, 64).half(), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: B.linear(x, w), lambda: B.matmul(named(blocks(6, 64)), w), lambda: grouped_matmul(x, experts, off)):
        with pytest.raises(ValueError, match="CUDA tensors"):     # refused for that alone
            call()


def test_sides_beyond_32_bits_are_refused():
    # (the packing of the C structure raised its own error there, and the library's for sides just above its limit)
    for most in (2 ** 31 - 1024, 2 ** 32 + 5):
        tall, wide = torch.zeros(1, 16).half().expand(most, 16), torch.zeros(16, 1).half().expand(16, most)
        huge, w = torch.zeros(1, 1, 16).half().expand(1, most, 16), torch.zeros(1, 8, 16).half()
        x, off, codes = torch.zeros(4, 16).half(), torch.tensor([0, 1], dtype=torch.int32), torch.zeros(1, 16).to(torch.float8_e4m3fn)
        for call in (lambda: B.linear(tall, w[0]),
                     lambda: B.linear(tall.expand(3, most, 16), w[0]),
                     lambda: B.linear(x, huge[0]),
                     lambda: B.quantize(tall),
                     lambda: B.quantize_both(wide, rows=128),
                     lambda: B.quantize(huge),
                     lambda: B.BlockFP8(codes.expand(most, 16), blocks(1, 16).scales),
                     lambda: grouped_matmul(tall, w, off),
                     lambda: grouped_matmul(x, huge, off)):
            with pytest.raises(ValueError, match="out of range"):
                call()
