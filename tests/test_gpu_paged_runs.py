"""GPU tests of one token's attention over caches so large that a wavefront takes
many stages of one sequence: loads into places that were read before, counted
waits over and over, pages looked up anew on the way."""

from __future__ import annotations

import pytest

from attention_reference import FP32, HALF, check, stored
from conftest import pkg
from test_gpu_kv_cache import index, make_table

pytestmark = pytest.mark.gpu


def dealt(lengths, kv_heads, dim, quantised):
    """(stages of a page look-up, tokens of a stage, [(sequence, first stage, stages)] of every
    wavefront's runs), by the kernel's rules for up to 16 heads a key head."""
    row = dim if quantised else 2 * dim
    pitch = max(128, 1 << (row - 1).bit_length())
    tokens = 32 if pitch >= 256 else 64
    lds = 2 * (2 * tokens * pitch + 128 * quantised)
    workers = 256 * min(4, 160 * 1024 // lds)
    chunks = [-(-n // tokens) for n in lengths]
    units = sum(chunks) * kv_heads
    starts = [units * w // workers for w in range(workers + 1)]
    runs, first, w = [], 0, 0
    for s, n in enumerate(chunks):
        for _ in range(kv_heads):
            end, at = first + n, first
            while at < end:
                while starts[w + 1] <= at:
                    w += 1
                upto = min(end, starts[w + 1])
                runs.append((s, at - first, upto - at))
                at = upto
            first = end
    return 1024 // tokens, tokens, runs


def cache_of(dev, lengths, kv_heads, dim, page_size, quantised, power=None):
    """Each of 16 query heads a key head finds nearly all of its weight at one token of its
    sequence, anywhere in it, so that every one of these tokens has to be the right one."""
    import torch

    M = pkg()
    g = torch.Generator(device=dev).manual_seed(7)
    pages = sum(-(-n // page_size) for n in lengths) + 3
    cache = M.KVCache(pages, page_size, kv_heads, dim, quantised=quantised, device=dev)
    for t in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales):
        if t is not None:
            t.view(torch.uint8).random_(0, 256, generator=g)
    table = make_table(dev, lengths, page_size, pages)
    offsets = [0]
    for n in lengths:
        offsets.append(offsets[-1] + n)
    k, v = (torch.randn(offsets[-1], kv_heads, dim, generator=g, device=dev).to(torch.bfloat16) for _ in range(2))
    if power is not None:
        v = ((1 + v.float().abs().fmod(0.75)) * 2.0**power).to(torch.bfloat16)
    q = torch.randn(len(lengths), kv_heads, 16, dim, generator=g, device=dev).to(torch.bfloat16)
    heads = torch.arange(kv_heads, device=dev)[:, None]
    for s, n in enumerate(lengths):
        at = torch.randint(n, (kv_heads, 16), generator=g, device=dev)
        k[offsets[s] + at, heads] = 3 * q[s]  # a score of 3 sqrt(dim), 24 or more: others' stay below 12
    cache.append(k, v, table, index([0] * len(lengths), dev), index(offsets, dev))
    return cache, table, k, v, offsets, q.view(len(lengths), 16 * kv_heads, dim)


def by_key_heads(q, k, v, offsets, quantised):
    """(result, bound) in 64 bits, all queries of a sequence and key head at once."""
    import torch

    k, v, q = stored(k, quantised), stored(v, quantised), q.double()
    group, scale = q.shape[1] // k.shape[1], q.shape[2] ** -0.5
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for s, (a, b) in enumerate(zip(offsets[:-1], offsets[1:])):
        for j in range(k.shape[1]):
            of, kk, vv = slice(j * group, (j + 1) * group), k[a:b, j].contiguous(), v[a:b, j].contiguous()
            p = (scale * (q[s, of] @ kk.t())).softmax(1)
            o, spread = p @ vv, p @ vv.abs()
            out[s, of], bound[s, of] = o, HALF * (spread + o.abs()) + FP32 * spread
    return out, bound


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dim, page_size", [(64, 16), (80, 64), (128, 16), (256, 1024)])
def test_many_stages_a_run(dev, dim, page_size, quantised):
    import torch

    ahead, tokens, _ = dealt([1], 1, dim, quantised)
    of = tokens / 64  # so that every width has runs of as many stages
    lengths = [int(n * of) for n in (40_000, 17, 31_234, 2000, 39_999, 24_000, 13_345, 1027, 16_500)]
    kv_heads = 8 if dim == 256 and not quantised else 16
    ahead, tokens, runs = dealt(lengths, kv_heads, dim, quantised)
    s, first, stages = max(runs, key=lambda r: r[2])
    assert stages > (2 * ahead if tokens == 64 else ahead + 2)
    cache, table, k, v, offsets, q = cache_of(dev, lengths, kv_heads, dim, page_size, quantised)
    got = cache.attend(q, table, index(lengths, dev))
    check(got, by_key_heads(q, k, v, offsets, quantised))
    assert torch.equal(cache.attend(q, table, index(lengths, dev)), got)
    # a bad page that only a later look-up of a run meets
    bad = (first + ahead + 1) * tokens // page_size
    assert bad * page_size < (first + stages) * tokens
    wrong = table.clone()
    wrong[s, bad] = -1
    other = [i for i in range(len(lengths)) if i != s]
    got_wrong = cache.attend(q, wrong, index(lengths, dev))
    assert bool(got_wrong[s].isnan().all()) and torch.equal(got_wrong[other], got[other])


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_stages_taken_again(dev, dim, quantised):
    """Values whose sums pass FP32's range: every run's second pass over its stages."""
    ahead, tokens, _ = dealt([1], 1, dim, quantised)
    lengths = [n * tokens // 64 for n in (40_000, 31_234, 2000, 39_999, 40_000, 17)]
    _, _, runs = dealt(lengths, 16, dim, quantised)
    assert max(r[2] for r in runs) > ahead + 2
    cache, table, k, v, offsets, q = cache_of(dev, lengths, 16, dim, 16, quantised, 126)
    check(cache.attend(q, table, index(lengths, dev)), by_key_heads(q, k, v, offsets, quantised))
