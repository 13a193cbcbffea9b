"""The C entry points of block-scaled FP8 and grouped products, without a GPU: every argument that a
kernel or the host arithmetic could not stand is refused before any of it runs."""
import pytest

from aeisu_b200 import _lib, build
from test_block_fp8 import HALF, packed


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
