"""GPU tests of the paged key-value cache: what is written and read back, bit
for bit, and one token's attention over it within the bounds of
attention_reference."""

from __future__ import annotations

import pytest

from attention_reference import FP32, HALF, check, stored
from conftest import pkg, submodule

pytestmark = pytest.mark.gpu


def index(values, dev):
    import torch

    return torch.tensor(values, dtype=torch.int32, device=dev)


def garbage(shape, kind, dev, seed=9):
    """Whatever memory holds, NaN among it."""
    import torch

    g = torch.Generator().manual_seed(seed)
    bits = torch.randint(0, 256, (*shape[:-1], shape[-1] * (1 if kind is torch.uint8 else 2)), generator=g, dtype=torch.uint8)
    return bits.to(dev) if kind is torch.uint8 else bits.to(dev).view(torch.bfloat16)


def make_cache(dev, pages, page_size, kv_heads, dim, quantised):
    import torch

    cache = pkg().KVCache(pages, page_size, kv_heads, dim, quantised=quantised, device=dev)
    for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
        t = getattr(cache, name)
        if t is not None:
            t.copy_(garbage(t.shape, t.dtype, dev))
    return cache


def make_table(dev, lengths, page_size, pages, spare=0, seed=3):
    """Pages in any order; entries past a sequence's last page are no pages."""
    import torch

    need = [-(-n // page_size) for n in lengths]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lengths), max([1, *need]) + spare), -7, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    assert at <= pages
    return table.to(dev)


def normal(dev, *shape, seed=0, std=1.0):
    import torch

    return (std * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(torch.bfloat16).to(dev)


def filled(dev, lengths, page_size, kv_heads, dim, quantised, spare_pages=2):
    """A cache that holds `lengths` tokens, its table, and the packed rows."""
    pages = sum(-(-n // page_size) for n in lengths) + spare_pages
    cache, table = make_cache(dev, pages, page_size, kv_heads, dim, quantised), make_table(dev, lengths, page_size, pages)
    total = sum(lengths)
    k, v = normal(dev, total, kv_heads, dim, seed=1), normal(dev, total, kv_heads, dim, seed=2)
    if dim >= 16:
        k[..., ::dim // 4] *= 3
    offsets = [0]
    for n in lengths:
        offsets.append(offsets[-1] + n)
    cache.append(k, v, table, index([0] * len(lengths), dev), index(offsets, dev))
    return cache, table, k, v, offsets


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dim", [16, 64, 80, 128, 208, 256])
@pytest.mark.parametrize("page_size", [16, 64])
def test_written_and_read_back(dev, quantised, dim, page_size):
    """Values come back as stored: the bf16 ones, or the nearest E4M3 code's."""
    import torch

    cache, table, k, v, offsets = filled(dev, [1, 16, 17, 0, 100], page_size, 3, dim, quantised)
    got = cache.read(table, index(offsets, dev), offsets[-1])
    for g, x in zip(got, (k, v)):
        assert torch.equal(g.double(), stored(x, quantised))


@pytest.mark.parametrize("sequences", [62, 63, 64, 4094, 4095, 5000])
def test_rows_of_many_sequences(dev, sequences):
    import torch

    lengths = torch.randint(0, 4, (sequences,), generator=torch.Generator().manual_seed(2)).tolist()
    cache, table, k, v, offsets = filled(dev, lengths, 16, 1, 16, False)
    got = cache.read(table, index(offsets, dev), offsets[-1] + 5)
    for rows, want in zip(got, (k, v)):
        assert torch.equal(rows[:-5], want) and not bool(rows[-5:].any())


@pytest.mark.parametrize("dim", [8, 24, 72, 136])
def test_bf16_rows_of_other_widths(dev, dim):
    import torch

    cache, table, k, v, offsets = filled(dev, [33, 5], 16, 2, dim, False)
    got = cache.read(table, index(offsets, dev), 38)
    assert torch.equal(got[0], k) and torch.equal(got[1], v)


def test_every_code_and_row_scale(dev):
    """Rows whose largest value lies at and around each power of two and each
    rounding border, down to the smallest and up to the largest bf16 numbers,
    and rows of zeros: codes, scales and values."""
    import torch

    dim = 64
    tops = []
    for e in (-133, -126, -118, -117, -109, -108, -107, -20, -1, 0, 1, 8, 9, 100, 126, 127):
        for m in (1.0, 1.0078125, 1.5, 1.7421875, 1.75, 1.7578125, 1.9921875):
            tops.append(m * 2.0**e)
    tops.append(0.0)
    top = torch.tensor(tops, dtype=torch.float64)
    ladder = torch.cat([torch.ones(1), -torch.ones(1), 2.0 ** -torch.linspace(0, 20, dim - 2)]).double()
    rows = (top[:, None] * ladder).to(torch.bfloat16)[:, None].to(dev)  # [n, 1, dim]
    n = rows.shape[0]
    cache = make_cache(dev, -(-n // 16), 16, 1, dim, True)
    table = make_table(dev, [n], 16, cache.k_pages.shape[0])
    cache.append(rows, -rows, table, index([0], dev), index([0, n], dev))
    k, v = cache.read(table, index([0, n], dev), n)
    want = stored(rows, True)
    assert torch.equal(k.double(), want) and torch.equal(v.double(), -want)
    # relative to the row's largest: half a step of the codes, or of the smallest one
    off, largest = (k.double() - rows.double()).abs(), rows.double().abs().amax(2, keepdim=True)
    smallest = torch.maximum(largest / 224 * 2.0**-10, torch.full_like(largest, 2.0**-127))
    assert bool((off <= torch.maximum(2.0**-4 * rows.double().abs(), smallest)).all())


def test_infinities_and_nans_are_stored_as_nan(dev):
    """... and the rest of their row as if they were not there."""
    import torch

    x = normal(dev, 20, 2, 64)
    wrong = x.clone()
    wrong[3, 0, 5], wrong[4, 1, 0], wrong[5, 0, 63] = float("inf"), float("-inf"), float("nan")
    zeroed = torch.where(wrong.isfinite(), wrong, torch.zeros_like(wrong))
    cache = make_cache(dev, 3, 16, 2, 64, True)
    table = make_table(dev, [20], 16, 3)
    cache.append(wrong, wrong, table, index([0], dev), index([0, 20], dev))
    k, v = cache.read(table, index([0, 20], dev), 20)
    assert torch.equal(k.isnan(), ~wrong.isfinite())
    assert torch.equal(torch.where(k.isnan(), 0, k).double(), stored(zeroed, True)) and torch.equal(k.isnan(), v.isnan())


@pytest.mark.parametrize("quantised", [False, True])
def test_only_the_new_places_change(dev, quantised):
    """Appending in chunks and one by one: every other byte of the cache stays,
    and what was there before is still read."""
    import torch

    lengths = [20, 0, 47]
    cache, table, k, v, offsets = filled(dev, lengths, 16, 2, 64, quantised, spare_pages=4)
    table = torch.cat([table, torch.full((3, 1), -1, dtype=torch.int32, device=dev)], 1)
    used = set(int(p) for p in table.flatten() if p >= 0)
    free = [p for p in range(cache.k_pages.shape[0]) if p not in used]
    table[1, 0] = free[0]
    names = [n for n in ("k_pages", "v_pages", "k_scales", "v_scales") if getattr(cache, n) is not None]
    before = {n: getattr(cache, n).clone() for n in names}
    new_k, new_v = normal(dev, 3, 2, 64, seed=5), normal(dev, 3, 2, 64, seed=6)
    cache.append(new_k, new_v, table, index(lengths, dev))
    touched = torch.zeros(cache.k_pages.shape[:3], dtype=torch.bool, device=dev)
    for s, n in enumerate(lengths):
        touched[int(table[s, n // 16]), :, n % 16] = True
    for n in names:
        now = getattr(cache, n)
        assert torch.equal(now[~touched].view(torch.uint8), before[n][~touched].view(torch.uint8)), n
    o = index([0, 21, 22, 70], dev)
    rk, rv = cache.read(table, o, 70)
    for got, old, new in ((rk, k, new_k), (rv, v, new_v)):
        want = torch.cat([old[:20], new[:1], new[1:2], old[20:], new[2:]])
        assert torch.equal(got.double(), stored(want, quantised))


def test_strided_rows_and_rows_of_no_sequence(dev):
    import torch

    joint = normal(dev, 40, 8, 64)
    q, k, v = joint.split([4, 2, 2], 1)
    cache = make_cache(dev, 4, 16, 2, 64, True)
    table = make_table(dev, [20, 10], 16, 4)
    before = cache.k_pages.clone()
    cache.append(k, v, table, index([0, 0], dev), index([5, 25, 35], dev))  # rows 0 .. 4 and 35 .. are nobody's
    rk, rv = cache.read(table, index([3, 23, 33], dev), 40)
    assert torch.equal(rk[3:33].double(), stored(k[5:35], True)) and torch.equal(rv[3:33].double(), stored(v[5:35], True))
    assert not rk[:3].any() and not rk[33:].any() and not rv[:3].any() and not rv[33:].any()
    places = torch.zeros(4, 16, dtype=torch.bool, device=dev)
    for s, n in ((0, 20), (1, 10)):
        for p in range(n):
            places[int(table[s, p // 16]), p % 16] = True
    kept = ~places[:, None, :].expand(4, 2, 16)
    assert torch.equal(cache.k_pages[kept], before[kept])


@pytest.mark.parametrize("quantised", [False, True])
def test_bad_pages(dev, quantised):
    """Pages outside the cache and positions past the table: nothing is
    written, reading gives NaN, attention NaN for that sequence alone."""
    import torch

    M = pkg()
    lengths = [40, 40, 40]
    cache, table, k, v, offsets = filled(dev, lengths, 16, 2, 64, quantised)
    q = normal(dev, 3, 4, 64, seed=7)
    clean = cache.attend(q, table, index(lengths, dev))
    for bad in (-1, cache.k_pages.shape[0], (1 << 31) - 1, -(1 << 31)):
        wrong = table.clone()
        wrong[1, 1] = bad
        got = cache.attend(q, wrong, index(lengths, dev))
        assert torch.equal(got[[0, 2]], clean[[0, 2]]) and got[1].isnan().all()
        rk, rv = cache.read(wrong, index(offsets, dev), 120)
        rows = torch.zeros(120, dtype=torch.bool, device=dev)
        rows[40 + 16:40 + 32] = True
        for got_rows, x in ((rk, k), (rv, v)):
            assert got_rows[rows].isnan().all()
            assert torch.equal(got_rows[~rows].double(), stored(x, quantised)[~rows])
        before = [t.clone() for t in (cache.k_pages, cache.v_pages)]
        cache.append(k[:1], v[:1], wrong[1:2], index([20], dev))
        cache.append(k[:1], v[:1], wrong[:1], index([48], dev))  # no fourth page
        cache.append(k[:1], v[:1], wrong[:1], index([-1], dev))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, (cache.k_pages, cache.v_pages)))
    # longer than the table, and negative lengths
    got = cache.attend(q, table, index([40, 49, -3], dev))
    assert torch.equal(got[0], clean[0]) and got[1].isnan().all() and not got[2].any()
    none = M.paged_attention(q, cache.k_pages, cache.v_pages, table[:, :0], index([0, 1, 0], dev), k_scales=cache.k_scales,
                             v_scales=cache.v_scales)
    assert not none[[0, 2]].any() and none[1].isnan().all()


# ------------------------------------------------------------- one token ---


def paged64(q, k, v, offsets, quantised, scale=None):
    """(result, bound) of one query a sequence over packed rows as stored."""
    import torch

    k, v, q = stored(k, quantised), stored(v, quantised), q.double()
    scale = q.shape[2] ** -0.5 if scale is None else scale
    group = q.shape[1] // k.shape[1]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    for s, (a, b) in enumerate(zip(offsets[:-1], offsets[1:])):
        if a == b:
            continue
        for h in range(q.shape[1]):
            p = (scale * (k[a:b, h // group] @ q[s, h])).softmax(0)
            vv = v[a:b, h // group]
            out[s, h] = p @ vv
            bound[s, h] = HALF * (p @ vv.abs() + out[s, h].abs()) + FP32 * (p @ vv.abs())
    return out, bound


def decode(dev, lengths, heads, kv_heads, dim, page_size, quantised, scale=None):
    cache, table, k, v, offsets = filled(dev, lengths, page_size, kv_heads, dim, quantised)
    q = normal(dev, len(lengths), heads, dim, seed=4)
    got = cache.attend(q, table, index(lengths, dev), scale=scale)
    check(got, paged64(q, k, v, offsets, quantised, scale))
    return cache, table, q, got


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("lengths", [[1], [2], [15], [16], [17], [31], [32], [33], [63], [64], [65], [127], [129], [255], [1000],
                                     [0], [0, 0, 5], [3, 0, 700, 1, 64], [40] * 70])
def test_lengths(dev, lengths, quantised):
    decode(dev, lengths, 8, 2, 128, 16, quantised)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dim", [16, 32, 64, 80, 96, 128, 144, 208, 256])
def test_widths(dev, dim, quantised):
    decode(dev, [1, 100, 37], 6, 2, dim, 32, quantised)


@pytest.mark.parametrize("dim", [8, 24, 72, 200, 248])
def test_widths_of_bf16_alone(dev, dim):
    decode(dev, [70, 5], 4, 2, dim, 16, False)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (3, 1), (8, 8), (15, 1), (16, 1), (17, 1), (32, 2), (40, 1), (96, 2)])
def test_head_groups(dev, heads, kv_heads, quantised):
    decode(dev, [90, 3], heads, kv_heads, 64, 16, quantised)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("page_size", [16, 32, 128, 1024, 65536])
def test_page_sizes(dev, page_size, quantised):
    decode(dev, [50, 1500, 17], 4, 1, 64, page_size, quantised)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_split_and_joined(dev, dim, quantised):
    """One sequence over the whole card, beside short ones; several workgroups' parts."""
    decode(dev, [30_000, 5, 1000], 8, 1, dim, 64, quantised)


def test_more_rows_than_the_fine_join_takes(dev):
    decode(dev, [3000, 1, 2000] + [70] * 30, 32, 4, 64, 16, False)


@pytest.mark.parametrize("sequences", [63, 64, 65, 129])
def test_many_sequences(dev, sequences):
    decode(dev, [(13 * i) % 90 for i in range(sequences)], 4, 2, 64, 16, True)


@pytest.mark.parametrize("sequences, heads, kv_heads, longest, long", [
    (130, 24, 1, 40, 0),  # two parts of a key head
    (300, 8, 8, 70, 0),  # more (sequence, head) parts than workers
    (1023, 1, 1, 5, 0), (1024, 1, 1, 5, 0), (1025, 1, 1, 5, 0),
    (1030, 2, 1, 20, 4000),  # one of them over many workers
    (4200, 1, 1, 3, 0),  # runs of more than 64 sequences
])
@pytest.mark.parametrize("quantised", [False, True])
def test_batches(dev, sequences, heads, kv_heads, longest, long, quantised):
    import torch

    lengths = torch.randint(0, longest + 1, (sequences,), generator=torch.Generator().manual_seed(sequences)).tolist()
    lengths[:3], lengths[-70:] = [0] * 3, [0] * 70  # starts and ends with sequences without a token
    if long:
        lengths[sequences // 2] = long
    decode(dev, lengths, heads, kv_heads, 64, 16, quantised)


@pytest.mark.parametrize("sequences", [3, 200, 1100])
def test_tables_without_a_page(dev, sequences):
    """0 where there is no token, NaN where there is one and no page."""
    import torch

    cache = make_cache(dev, 2, 16, 2, 80, False)
    lengths = torch.arange(sequences, dtype=torch.int32) % 3
    got = cache.attend(normal(dev, sequences, 6, 80), torch.zeros(sequences, 0, dtype=torch.int32, device=dev), lengths.to(dev)).cpu()
    assert bool((got[lengths == 0] == 0).all()) and bool(got[lengths > 0].isnan().all())


@pytest.mark.parametrize("scale", [1e-3, 1.0])
def test_scales(dev, scale):
    decode(dev, [100, 40], 4, 2, 64, 16, True, scale)


def test_is_what_packed_attention_gives_the_last_query(dev):
    """Both forms of one formula, each within its bound of the other."""
    import torch

    M = pkg()
    lengths = [130, 64, 1]
    cache, table, k, v, offsets = filled(dev, lengths, 16, 2, 128, False)
    q = normal(dev, 3, 8, 128, seed=4)
    got = cache.attend(q, table, index(lengths, dev))
    packed = M.packed_attention(q, k, v, index([0, 1, 2, 3], dev), index(offsets, dev))
    want, bound = paged64(q, k, v, offsets, False)
    assert bool(((got.double() - packed.double()).abs() <= 2.04 * bound + 2.0**-133).all())


def test_what_lies_behind_the_last_token_does_not_matter(dev):
    """Infinities and NaN in the rest of a page, in other pages, in scales."""
    import torch

    for quantised in (False, True):
        cache, table, k, v, offsets = filled(dev, [37, 81], 32, 2, 64, quantised)
        q = normal(dev, 2, 4, 64, seed=4)
        want = cache.attend(q, table, index([37, 81], dev))
        owned = torch.zeros(cache.k_pages.shape[0], 32, dtype=torch.bool, device=dev)
        for s, n in ((0, 37), (1, 81)):
            for p in range(n):
                owned[int(table[s, p // 32]), p % 32] = True
        rest = ~owned[:, None].expand(-1, 2, 32)
        for fill in ((0x7F, 0xFF, 0x00, 0x80) if quantised else (float("nan"), float("inf"), -float("inf"), 1e30)):
            for t in (cache.k_pages, cache.v_pages):
                t[rest] = fill
            for t in (cache.k_scales, cache.v_scales):
                if t is not None:
                    t[rest] = 255
            assert torch.equal(cache.attend(q, table, index([37, 81], dev)), want), fill


def test_shared_pages_strided_queries_and_tables(dev):
    """Two sequences with the same first pages; q as a slice of a joint tensor, a
    table that is a slice of a wider one."""
    import torch

    cache, table, k, v, offsets = filled(dev, [64, 100], 16, 2, 64, True)
    shared = torch.stack([table[1], table[1]])
    joint = normal(dev, 2, 8, 64, seed=4)
    q = joint[:, 2:6]
    wide = torch.full((2, 40), -1, dtype=torch.int32, device=dev)
    wide[:, 3:3 + shared.shape[1]] = shared
    got = cache.attend(q, wide[:, 3:3 + shared.shape[1]], index([100, 33], dev))
    rows_k, rows_v = torch.cat([k[64:], k[64:97]]), torch.cat([v[64:], v[64:97]])
    check(got, paged64(q, rows_k, rows_v, [0, 100, 133], True))
    across = shared.t().contiguous().t()  # column by column
    assert torch.equal(cache.attend(q, across, index([100, 33], dev)), got)


def test_same_bits_every_time(dev):
    import torch

    cache, table, q, first = decode(dev, [5000, 300, 77], 8, 2, 128, 16, True)
    for _ in range(3):
        assert torch.equal(cache.attend(q, table, index([5000, 300, 77], dev)), first)


def test_offsets_past_32_bits(dev):
    """Pages that lie past 2^32 bytes and elements of the cache."""
    import torch

    M = pkg()
    pages, shape = 70_000, (8, 64, 128)  # 9 GB of keys in bf16, 4.6e9 elements
    k_pages = torch.empty((pages, *shape), dtype=torch.bfloat16, device=dev)
    v_pages = torch.empty_like(k_pages)
    k, v = normal(dev, 150, 8, 128, seed=1), normal(dev, 150, 8, 128, seed=2)
    table = index([[pages - 1, 5, pages - 7]], dev)
    M.append_kv(k, v, k_pages, v_pages, table, index([0], dev), index([0, 150], dev))
    rk, rv = M.read_kv(k_pages, v_pages, table, index([0, 150], dev), 150)
    assert torch.equal(rk, k) and torch.equal(rv, v)
    q = normal(dev, 1, 16, 128, seed=4)
    check(M.paged_attention(q, k_pages, v_pages, table, index([150], dev)), paged64(q, k, v, [0, 150], False))


def test_captured_step_whose_lengths_and_tables_change(dev):
    """Append and attention in one graph, replayed as sequences grow, with eager
    work between: every replay is the eager step."""
    import torch

    M = pkg()
    caches = [make_cache(dev, 30, 16, 2, 64, True) for _ in range(2)]
    for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
        getattr(caches[1], name).copy_(getattr(caches[0], name))
    table = torch.stack([torch.arange(10), torch.arange(10, 20), torch.arange(20, 30)]).to(torch.int32).to(dev)
    state = [normal(dev, 3, 4, 64), normal(dev, 3, 2, 64), normal(dev, 3, 2, 64), index([0, 0, 0], dev), index([1, 1, 1], dev), table.clone()]

    def step(cache, q, k, v, before, after, pages):
        cache.append(k, v, pages, before)
        return cache.attend(q, pages, after)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step(caches[0], *state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step(caches[0], *state)
    step(caches[1], *state)
    for n in range(1, 60, 7):
        lengths = [n, 2 * n, 0 if n % 2 else 5]
        pages = table.roll(n, 0) if n > 30 else table
        new = [normal(dev, 3, 4, 64, seed=n), normal(dev, 3, 2, 64, seed=n + 100), normal(dev, 3, 2, 64, seed=n + 200),
               index(lengths, dev), index([x + 1 for x in lengths], dev), pages]
        for s, t in zip(state, new):
            s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = step(caches[1], *new)
        assert torch.equal(out.nan_to_num(9), want.nan_to_num(9)), n


def test_two_streams_at_once(dev):
    import torch

    sets = [decode(dev, [9000, 40], 8, 2, 128, 16, True), decode(dev, [100, 7000, 3], 16, 4, 128, 64, False)]
    lengths = [index([9000, 40], dev), index([100, 7000, 3], dev)]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, ((cache, table, q, _), stream) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(stream):
                got[i].append(cache.attend(q, table, lengths[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, s[3]) for s, each in zip(sets, got) for g in each)


def test_as_custom_ops(dev):
    import torch

    M = pkg()
    cache, table, q, want = decode(dev, [50, 20], 4, 2, 64, 16, True)
    tensors = (cache.k_pages, cache.v_pages, table)
    got = torch.ops.glm53.paged_attention(q, *tensors, index([50, 20], dev), cache.k_scales, cache.v_scales, 0.125)
    assert torch.equal(got, want)
    torch.library.opcheck(torch.ops.glm53.paged_attention.default,
                          (q, *tensors, index([50, 20], dev), cache.k_scales, cache.v_scales, 0.125))
    torch.library.opcheck(torch.ops.glm53.read_kv.default,
                          (*tensors, index([0, 50, 70], dev), 70, cache.k_scales, cache.v_scales))
    k = normal(dev, 2, 2, 64)

    def step(k, q):
        M.append_kv(k, k, cache.k_pages, cache.v_pages, table, index([49, 19], dev), k_scales=cache.k_scales, v_scales=cache.v_scales)
        return M.paged_attention(q, cache.k_pages, cache.v_pages, table, index([50, 20], dev), k_scales=cache.k_scales,
                                 v_scales=cache.v_scales)

    eager = step(k, q)
    assert torch.equal(torch.compile(step, backend="eager")(k, q), eager)


def test_python_refusals(dev):
    import torch

    M = pkg()
    cache = pkg().KVCache(4, 16, 2, 64, device=dev)
    q8 = pkg().KVCache(4, 16, 2, 64, quantised=True, device=dev)
    table, lengths = torch.zeros(3, 2, dtype=torch.int32, device=dev), torch.ones(3, dtype=torch.int32, device=dev)
    q, k = normal(dev, 3, 4, 64), normal(dev, 3, 2, 64)
    P = (cache.k_pages, cache.v_pages)
    attends = [
        (q.float(), *P, table, lengths), (q[:2], *P, table, lengths), (q[:, :3], *P, table, lengths), (q[..., :32], *P, table, lengths),
        (q, P[0], P[1][:3], table, lengths), (q, P[0], P[1].float(), table, lengths), (q, P[0].transpose(1, 2), P[1].transpose(1, 2), table, lengths),
        (q, *P, table.long(), lengths), (q, *P, table[0], lengths), (q, *P, table, lengths.long()), (q, *P, table, lengths[:2]),
        (q, q8.k_pages, q8.v_pages, table, lengths), (q, *P, table.cpu(), lengths), (q, *P, table, lengths.cpu()),
        (q, P[0][:, :, :8].contiguous(), P[1][:, :, :8].contiguous(), table, lengths), (q, P[0][:0], P[1][:0], table, lengths),
    ]
    for args in attends:
        with pytest.raises((ValueError, RuntimeError)):
            M.paged_attention(*args)
    with pytest.raises(ValueError, match="belong"):
        M.paged_attention(q, *P, table, lengths, k_scales=q8.k_scales, v_scales=q8.v_scales)
    with pytest.raises(ValueError, match="uint8"):
        M.paged_attention(q, q8.k_pages, q8.v_pages, table, lengths, k_scales=q8.k_scales[:3], v_scales=q8.v_scales)
    for scale in (0.0, -2.0, float("nan")):
        with pytest.raises(ValueError, match="scale"):
            M.paged_attention(q, *P, table, lengths, scale=scale)
    o = index([0, 1, 2, 3], dev)
    for args in [(k[:2], k[:2], *P, table, lengths), (k, k[:2], *P, table, lengths), (q, q, *P, table, lengths), (k.float(), k, *P, table, lengths),
                 (k, k, *P, table, lengths, o[:3]), (k, k, *P, table, lengths, o.long()), (k, k, *P, table, lengths[:1])]:
        with pytest.raises(ValueError):
            M.append_kv(*args)
    for args in [(*P, table, o[:3], 3), (*P, table, None, 3), (*P, table, o, -1), (*P, table, o.long(), 3)]:
        with pytest.raises((ValueError, RuntimeError)):
            M.read_kv(*args)
    assert M.read_kv(*P, table, o, 0)[0].shape == (0, 2, 64)
    assert M.paged_attention(q[:0], *P, table[:0], lengths[:0]).shape == (0, 4, 64)
    M.append_kv(k[:0], k[:0], *P, table[:0], lengths[:0])
