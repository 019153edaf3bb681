"""GPU tests of attention over values near the ends of FP32: a mean of finite
values is finite, whatever the sum of the weights that it is made of."""

from __future__ import annotations

import pytest

from attention_reference import attention64, check
from conftest import pkg
from test_gpu_attention import gradients, index, inputs, offsets_of

pytestmark = pytest.mark.gpu


def large(t, power):
    """Positive bf16 values from 2^power to 2^(power + 1)."""
    import torch

    return ((1 + t.float().abs().fmod(1)) * 2.0**power).to(torch.bfloat16)


@pytest.mark.parametrize("keys, value", [(64, 1e37), (4096, 1e35), (1, 3e38), (3, 3e38)])
@pytest.mark.parametrize("dim", [64, 128])
def test_equal_values(dev, keys, value, dim):
    """Equal keys and values: the result is the value, by one rounding of each weight
    and one of the result."""
    import torch

    q, k, v, _ = inputs(dev, keys, keys, 2, 1, dim)
    k[:], v[:] = k[0], value
    got = pkg().packed_attention(q, k, v, causal=False)
    want = v[0, 0, 0].double()
    assert bool(((got.double() - want).abs() <= 2 * 2.0**-8 * want).all())


@pytest.mark.parametrize("dim", [64, 72, 128, 200, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_large_values_and_their_gradients(dev, dim, causal):
    """Sums of weights times values pass 2^128, means do not; d_out of 2^-100 keeps
    the gradients in range."""
    lengths = [300, 1, 70]
    o = offsets_of(lengths)
    q, k, v, d_out = inputs(dev, o[-1], o[-1], 4, 2, dim)
    v, d_out = large(v, 121), d_out * 2.0**-97
    got = gradients(q, k, v, d_out, index(o, dev), causal=causal)
    want = attention64(q, k, v, o, o, causal, None, d_out)
    for name in got:
        check(got[name], want[name], name)


def test_weights_above_one(dev):
    """Maxima that grow slowly from key to key, so that weights reach 2^8 of the one that is kept."""
    import torch

    q, k, v, _ = inputs(dev, 512, 512, 1, 1, 64)
    q[:], k[:] = 1, 0
    k[:, 0, 0] = torch.linspace(0, 60, 512, device=dev)  # scores up to 7.5: 2^10.8
    v = large(v, 125)
    got = pkg().packed_attention(q, k, v, causal=False)
    check(got, attention64(q, k, v, [0, 512], [0, 512], False)["out"])


def test_rows_and_columns_beside_large_ones_keep_their_bits(dev):
    """A tile's rows that stay in range, and a row's columns, have the bits of a call without the others."""
    import torch

    q, k, v, _ = inputs(dev, 200, 200, 2, 1, 64)
    M = pkg()
    want = M.packed_attention(q, k, v)
    w = v.clone()
    w[:, :, 1:] = large(v, 124)[:, :, 1:]
    got = M.packed_attention(q, k, w)
    assert bool(got.isfinite().all()) and torch.equal(got[..., 0], want[..., 0])
    few = M.packed_attention(q[:5], k[:5], w[:5])  # sums of at most 5 * 2^125
    assert torch.equal(got[:5], few)
    # a masked NaN beside them
    w[150] = float("nan")
    again = M.packed_attention(q, k, w)
    assert torch.equal(again[:150], got[:150]) and bool(again[150:].isnan().all())


@pytest.mark.parametrize("causal", [True, False])
def test_scores_that_no_number_holds(dev, causal):
    """Scaled scores past FP32's range give NaN, of results and of what they reach, not 0."""
    q, k, v, d_out = inputs(dev, 150, 150, 2, 1, 64)
    want = gradients(q, k, v, d_out, index([0, 60, 150], dev), causal=causal, scale=4.0)
    q, k = q.clone(), k.clone()
    q[70, 1], k[60:62, 0] = 2.0**60, 2.0**61  # 2^127 of scores, which are numbers
    got = gradients(q, k, v, d_out, index([0, 60, 150], dev), causal=causal, scale=4.0)
    assert bool(got["out"][70, 1].isnan().all()) and bool(got["d_q"][70, 1].isnan().all())
    assert bool(got["d_k"][60].isnan().all()) and bool(got["d_v"][60].isnan().all())
    for name in got:  # the other sequence
        assert (got[name][:60] == want[name][:60]).all(), name
