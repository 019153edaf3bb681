"""CPU checks of attention's limits: the scales that are refused."""

from __future__ import annotations

import pytest

from conftest import submodule
from test_attention_refusals import _attention, _cache, _paged


@pytest.mark.parametrize("scale", [2.0**127 * 1.5, 2.0**127 * (1 + 2.0**-23), 2.0**-65])
def test_scales_without_a_finite_logarithm(scale):
    """Weights are 2^(scale log2(e) score): the factor has to be an FP32 number."""
    N = submodule("_native")
    lib = N.load_library()
    for call in (lambda: lib.glm53_packed_attention(_attention(N, scale=scale), None),
                 lambda: lib.glm53_packed_attention_backward(_attention(N, scale=scale), None),
                 lambda: _paged(N, lib, _cache(N), scale=scale)):
        assert call() == N.INVALID_ARGUMENT
        assert "scale" in lib.glm53_last_error().decode()
    with pytest.raises(ValueError, match="scale"):
        submodule("attention").check_scale(scale, 64)


@pytest.mark.parametrize("scale", [2.0**127, 2.0**-64, None])
def test_scales_that_are_taken(scale):
    A = submodule("attention")
    assert A.check_scale(scale, 64) == (0.125 if scale is None else scale)
    N = submodule("_native")
    empty = _attention(N, tokens=0, out=None, q=N.HeadRows(None, 0, 0), scale=0.125 if scale is None else scale)
    assert N.load_library().glm53_packed_attention(empty, None) == N.OK
