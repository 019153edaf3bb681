"""GPU tests of gradients where both rules meet: as many keys and key heads as 128
keys a workgroup take, and few enough that the rows are split over workgroups."""

from __future__ import annotations

import pytest

from attention_reference import attention64, check
from conftest import submodule
from test_gpu_attention import gradients, index, inputs, offsets_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths, heads, kv_heads, dim", [
    ([4096], 8, 8, 64), ([4096], 16, 8, 64), ([2500, 0, 1596], 24, 8, 64), ([2048], 32, 16, 56), ([8100], 8, 4, 64), ([8192], 4, 4, 64),
])
def test_wide_tiles_in_parts(dev, lengths, heads, kv_heads, dim):
    """All heads of a key head, some rows of no sequence where lengths end before the tensors."""
    import torch

    tokens = 32_768 // kv_heads
    size = submodule("_native").lib().glm53_packed_attention_backward_split_bytes
    assert size(tokens, tokens, len(lengths), heads, kv_heads, dim) == 2 * 8 * 32_768 * dim  # two parts
    o = offsets_of(lengths)
    q, k, v, d_out = inputs(dev, tokens, tokens, heads, kv_heads, dim)
    got = gradients(q, k, v, d_out, index(o, dev), causal=False)
    again = gradients(q, k, v, d_out, index(o, dev), causal=False)
    group = heads // kv_heads
    for j in (0, kv_heads - 1):
        of, at = slice(j * group, (j + 1) * group), slice(j, j + 1)
        want = attention64(q[:, of], k[:, at], v[:, at], o, o, False, None, d_out[:, of])
        for name in got:
            check(got[name][:, at if name in ("d_k", "d_v") else of], want[name], name)
    for name in got:
        assert torch.equal(got[name], again[name]) and not bool(got[name][o[-1]:].any()), name


def test_wide_tiles_in_parts_and_infinities(dev):
    """An infinity in a row of one part reaches its column of every key of the sequence, and no other sequence."""
    import torch

    q, k, v, d_out = inputs(dev, 4096, 4096, 16, 8, 64)
    o = index([0, 3000, 4096], dev)
    want = gradients(q, k, v, d_out, o, causal=False)
    d_out[2900, 1, 3] = float("inf")
    got = gradients(q, k, v, d_out, o, causal=False)
    assert not bool(got["d_v"][:3000, 0, 3].isfinite().any())
    rest = [c for c in range(64) if c != 3]
    assert torch.equal(got["d_v"][:, 0, rest], want["d_v"][:, 0, rest])
    for name in ("d_k", "d_v"):
        assert torch.equal(got[name][3000:], want[name][3000:]) and torch.equal(got[name][:, 1:], want[name][:, 1:])
