"""GPU tests of one token's attention over cached values near the ends of FP32:
a mean of finite values is finite, in one part, in several, and where they join."""

from __future__ import annotations

import pytest

from attention_reference import check
from conftest import pkg
from test_gpu_kv_cache import index, make_cache, make_table, normal, paged64

pytestmark = pytest.mark.gpu


def cached(dev, lengths, k, v, page_size, quantised):
    pages = sum(-(-n // page_size) for n in lengths) + 2
    cache = make_cache(dev, pages, page_size, k.shape[1], k.shape[2], quantised)
    table = make_table(dev, lengths, page_size, pages)
    offsets = [0]
    for n in lengths:
        offsets.append(offsets[-1] + n)
    cache.append(k, v, table, index([0] * len(lengths), dev), index(offsets, dev))
    return cache, table, offsets


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
@pytest.mark.parametrize("power", [120, 126])
def test_large_values(dev, dim, power, quantised):
    """Values from 2^power to 1.75 * 2^power (240 * 2^120 is the largest of a code): of 2^126 a few
    tokens' sum passes 2^128, of 2^120 only that of many parts."""
    import torch

    lengths = [1, 5, 100, 3000, 0, 30_000]
    total = sum(lengths)
    k, v = normal(dev, total, 1, dim, seed=1), normal(dev, total, 1, dim, seed=2)
    v = ((1 + v.float().abs().fmod(0.75)) * 2.0**power).to(torch.bfloat16)
    cache, table, offsets = cached(dev, lengths, k, v, 16, quantised)
    q = normal(dev, len(lengths), 8, dim, seed=4)
    check(cache.attend(q, table, index(lengths, dev)), paged64(q, k, v, offsets, quantised))


@pytest.mark.parametrize("quantised", [False, True])
def test_some_parts_large(dev, quantised):
    """Large values in a few tokens of many: parts in range beside parts that are not, both signs."""
    import torch

    lengths = [20_000, 700]
    k, v = normal(dev, 20_700, 2, 64, seed=1), normal(dev, 20_700, 2, 64, seed=2)
    for at in (range(100, 400), range(12_000, 12_064), range(20_100, 20_400)):
        v[at] = (v[at].sign() * 2.0**126).to(torch.bfloat16)
    v[150:350] = 2.0**126
    cache, table, offsets = cached(dev, lengths, k, v, 64, quantised)
    q = normal(dev, 2, 6, 64, seed=4)
    check(cache.attend(q, table, index(lengths, dev)), paged64(q, k, v, offsets, quantised))


def test_zero_codes_of_large_rows(dev):
    """Rows whose power of two is the largest, and zeros among their codes: the last
    tokens' weights are 255.9 of the first ones', whose maximum is kept."""
    import torch

    k, v = (torch.zeros(40, 1, 64, dtype=torch.bfloat16, device=dev) for _ in range(2))
    k[32:, 0, :3] = torch.tensor([44, 0.34375, 0.015625], device=dev)  # codes: 8 * 7.9997 / log2(e)
    v[:, 0, ::2] = 3e38
    cache, table, offsets = cached(dev, [40], k, v, 16, True)
    q = torch.ones(1, 2, 64, dtype=torch.bfloat16, device=dev)
    got = cache.attend(q, table, index([40], dev))
    check(got, paged64(q, k, v, offsets, True))
    assert not bool(got[..., 1::2].any())


@pytest.mark.parametrize("quantised", [False, True])
def test_other_heads_keep_their_bits(dev, quantised):
    """Large values of one key head, and of one sequence, change no other one's results."""
    import torch

    lengths = [9000, 50]
    k, v = normal(dev, 9050, 2, 64, seed=1), normal(dev, 9050, 2, 64, seed=2)
    q = normal(dev, 2, 4, 64, seed=4)
    cache, table, _ = cached(dev, lengths, k, v, 16, quantised)
    want = cache.attend(q, table, index(lengths, dev))
    v[:9000, 1] = 2.0**126
    cache, table, _ = cached(dev, lengths, k, v, 16, quantised)
    got = cache.attend(q, table, index(lengths, dev))
    assert torch.equal(got[1], want[1]) and torch.equal(got[0, :2], want[0, :2])
    assert bool(((got[0, 2:].double() - 2.0**126).abs() <= 2 * 2.0**-8 * 2.0**126).all())


@pytest.mark.parametrize("lengths", [[1], [50], [20_000]])
def test_scores_that_no_number_holds(dev, lengths):
    """Scaled scores past FP32's range give NaN, not 0: in one part, and joined."""
    n = lengths[0]
    k, v = normal(dev, n, 1, 64, seed=1), normal(dev, n, 1, 64, seed=2)
    k[n // 2] = 2.0**60
    cache, table, _ = cached(dev, lengths, k, v, 16, False)
    q = normal(dev, 1, 2, 64, seed=4)
    q[0, 1] = 2.0**60
    got = cache.attend(q, table, index(lengths, dev), scale=4.0)  # of 2^126
    assert bool(got[0, 1].isnan().all())
