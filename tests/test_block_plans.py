"""CPU checks of the plans of the dense block's products, read from the sizes
of their workspaces."""

from __future__ import annotations

import pytest

from conftest import submodule


@pytest.fixture(scope="module")
def libso():
    return submodule("_native").load_library()


def _cdiv(a, b):
    return -(-a // b)


def _used(steps, parts):
    """Parts of a contraction of `steps` steps that have one."""
    return _cdiv(steps, _cdiv(steps, parts))


@pytest.mark.parametrize("rows", [1, 16])
@pytest.mark.parametrize("hidden, inter", [(1024, 896), (512, 896), (1536, 896), (1024, 1664), (2048, 640)])
def test_no_part_of_an_input_gradient_is_empty(libso, rows, hidden, inter):
    """Up to 16 rows the gradient of x is one contraction over four segments:
    high and low parts of dG and dU, in 64 x 128 tiles with steps of 128."""
    plane = 2 * 2 * rows * inter
    free = libso.glm53_gated_mlp_backward_workspace_bytes(rows, hidden, inter) - 2 * _cdiv(plane, 256) * 256
    parts, rest = divmod(free, 4 * rows * hidden)  # the largest of the products' partial results
    assert rest == 0 and parts > 1
    assert _used(4 * _cdiv(inter, 128), parts) == parts


@pytest.mark.parametrize("rows, n, k", [(64, 264, 4224), (33, 512, 4224), (128, 200, 2176), (64, 520, 8320), (100, 72, 5248)])
def test_no_part_of_a_4_bit_product_is_empty(libso, rows, n, k):
    parts, rest = divmod(libso.glm53_int4_linear_workspace_bytes(rows, n, k), 4 * rows * _cdiv(n, 4) * 4)
    assert rest == 0 and parts > 1
    assert _used(_cdiv(k, 128), parts) == parts
