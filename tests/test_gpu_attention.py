"""GPU tests of attention over packed sequences and its gradients, element by
element against 64 bits within the bounds of attention_reference."""

from __future__ import annotations

import pytest

from attention_reference import attention64, check
from conftest import pkg, submodule

pytestmark = pytest.mark.gpu


def offsets_of(lengths, start=0):
    got = [start]
    for n in lengths:
        got.append(got[-1] + n)
    return got


def index(values, dev):
    import torch

    return torch.tensor(values, dtype=torch.int32, device=dev)


def inputs(dev, tokens, keys, heads, kv_heads, dim, seed=0):
    import torch

    g = torch.Generator().manual_seed(seed)

    def normal(*shape, std=1.0):
        return (std * torch.randn(shape, generator=g)).to(torch.bfloat16).to(dev)

    q, k, v = normal(tokens, heads, dim), normal(keys, kv_heads, dim), normal(keys, kv_heads, dim)
    if dim >= 16:
        k[..., ::dim // 4] *= 3  # a few wide channels
    return q, k, v, normal(tokens, heads, dim, std=0.1)


def gradients(q, k, v, d_out, *args, **kw):
    import torch

    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = pkg().packed_attention(q, k, v, *args, **kw)
    return dict(zip(("out", "d_q", "d_k", "d_v"), (out.detach(), *torch.autograd.grad(out, [q, k, v], d_out))))


def run(dev, queries, keys, heads, kv_heads, dim, causal, seed=0, scale=None):
    """The forward call alone, and with gradients, against 64 bits."""
    import torch

    oq, ok = offsets_of(queries), offsets_of(keys)
    q, k, v, d_out = inputs(dev, oq[-1], ok[-1], heads, kv_heads, dim, seed)
    args = (index(oq, dev), index(ok, dev) if keys != queries else None)
    got = gradients(q, k, v, d_out, *args, causal=causal, scale=scale)
    with torch.no_grad():
        assert torch.equal(pkg().packed_attention(q, k, v, *args, causal=causal, scale=scale), got["out"])
    want = attention64(q, k, v, oq, ok, causal, scale, d_out)
    for name in got:
        check(got[name], want[name], name)
    return q, k, v, d_out, args, got


@pytest.mark.parametrize("dim", [8, 32, 64, 72, 96, 128, 136, 200, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_widths(dev, dim, causal):
    run(dev, [37, 1, 130], [37, 1, 130], 6, 2, dim, causal)


@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (3, 1), (4, 4), (10, 2), (7, 1), (16, 1), (24, 2), (40, 8)])
def test_head_groups(dev, heads, kv_heads):
    run(dev, [70, 65], [70, 65], heads, kv_heads, 64, True)


@pytest.mark.parametrize("lengths", [[1], [2], [31], [32], [33], [63], [64], [65], [127], [128], [129], [191], [192], [193], [500],
                                     [1, 1, 1, 1], [64, 64], [63, 1, 64, 200], [0, 5, 0, 0, 7, 0], [300, 0, 1], [129, 127, 128]])
@pytest.mark.parametrize("dim", [64, 128])
def test_lengths(dev, lengths, dim):
    run(dev, lengths, lengths, 4, 2, dim, True)


@pytest.mark.parametrize("queries, keys", [
    ([1, 1], [1, 100]), ([5], [300]), ([64, 3], [128, 3]), ([10, 0, 4], [100, 7, 64]),
    ([30, 50], [10, 20]),      # more queries than keys: the first ones see none
    ([40, 9], [0, 60]), ([65], [64]), ([200], [1]), ([129, 130], [64, 500]),
])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_of_another_length(dev, queries, keys, causal):
    run(dev, queries, keys, 6, 2, 64, causal)
    run(dev, queries, keys, 3, 3, 128, causal)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_longer(dev, dim, causal):
    """Many tiles a sequence, and key tiles of 64 and of 128 keys."""
    run(dev, [1100, 900], [1100, 900], 4, 2, dim, causal)


@pytest.mark.parametrize("queries, keys, heads, kv_heads, dim, causal", [
    ([3000], [3000], 8, 1, 128, True), ([2900, 0, 350], [2900, 0, 350], 8, 1, 64, True), ([2900], [2900], 8, 1, 96, False),
    ([1500], [1500], 8, 2, 256, True), ([1500], [1500], 8, 2, 200, False), ([5000], [70], 6, 2, 128, False),
    ([5000], [70], 6, 2, 128, True), ([600, 2500], [2600, 500], 5, 1, 128, True),
])
def test_gradients_of_few_keys(dev, queries, keys, heads, kv_heads, dim, causal):
    """The rows of a tile of keys are split, and the parts added; every subset of
    gradients alone has the joint call's bits."""
    import torch

    N = submodule("_native")
    size = N.lib().glm53_packed_attention_backward_split_bytes
    assert size(sum(queries), sum(keys), len(queries), heads, kv_heads, dim) > 0
    q, k, v, d_out, args, got = run(dev, queries, keys, heads, kv_heads, dim, causal)
    A = submodule("attention")
    out, lse = A.native_packed_attention(q, k, v, *args, causal, dim**-0.5, True)

    def gradients_of(wanted):
        return A.native_packed_attention_backward(q, k, v, *args, out, lse, d_out, causal, dim**-0.5, wanted)

    for wanted in ([False, True, False], [False, False, True], [False, True, True]):
        for g, name in zip(gradients_of(wanted), ("d_q", "d_k", "d_v")):
            assert g is None or torch.equal(g, got[name]), (wanted, name)


def test_without_the_workspace_of_parts(dev):
    """The native call with the least workspace does not split, and is right too."""
    import ctypes

    import torch

    A, N = submodule("attention"), submodule("_native")
    q, k, v, d_out = inputs(dev, 2000, 2000, 8, 1, 128)
    out, lse = A.native_packed_attention(q, k, v, None, None, True, 128**-0.5, True)
    d, alive = A._descriptor(q, k, v, None, None, out, lse, True, 128**-0.5)
    d_out, d.d_out = A.head_rows(d_out)
    got = {"d_q": torch.empty_like(q), "d_k": torch.empty_like(k), "d_v": torch.empty_like(v)}
    d.d_q, d.d_k, d.d_v = (t.data_ptr() for t in got.values())
    least = N.lib().glm53_packed_attention_backward_workspace_bytes(2000, 8)
    assert N.lib().glm53_packed_attention_backward_split_bytes(2000, 2000, 0, 8, 1, 128) > 0
    guarded = torch.full((least + 4096,), 77, dtype=torch.uint8, device=dev)
    d.workspace, d.workspace_bytes = guarded.data_ptr(), least
    N.run(q.get_device(), N.lib().glm53_packed_attention_backward, ctypes.byref(d))
    want = attention64(q, k, v, [0, 2000], [0, 2000], True, None, d_out)
    for name in got:
        check(got[name], want[name], name)
    assert bool((guarded[least:] == 77).all())


def test_parts_and_infinities(dev):
    """An infinity in a row of one part reaches the keys that the row sees, and no other."""
    import torch

    q, k, v, d_out = inputs(dev, 3000, 3000, 4, 1, 64)
    want = gradients(q, k, v, d_out)
    d_out[1500, 1, 3] = float("inf")
    got = gradients(q, k, v, d_out)
    assert bool(got["d_v"][:1501, 0, 3].isinf().all())
    for name in ("d_k", "d_v"):
        assert torch.equal(got[name][1501:], want[name][1501:])


@pytest.mark.parametrize("dim, causal, heads, tokens", [(128, False, 8, 4200), (64, False, 8, 4200), (96, False, 8, 4200),
                                                        (128, True, 32, 2100), (64, True, 32, 2100)])
def test_wide_key_tiles(dev, dim, causal, heads, tokens):
    """As many keys and key heads as the kernel of 128 keys a workgroup takes,
    in sequences of different lengths, against the sums of pieces that the other
    one makes of each sequence's key heads."""
    import torch

    lengths = [tokens // 2, tokens // 3, tokens - tokens // 2 - tokens // 3]
    o = offsets_of(lengths)
    q, k, v, d_out = inputs(dev, tokens, tokens, heads, heads, dim)
    got = gradients(q, k, v, d_out, index(o, dev), causal=causal)
    few = 2
    parts = [gradients(q[:, h:h + few], k[:, h:h + few], v[:, h:h + few], d_out[:, h:h + few], index(o, dev), causal=causal)
             for h in range(0, heads, few)]
    for name in got:
        joined = torch.cat([p[name] for p in parts], 1)
        if name in ("out", "d_q"):
            assert torch.equal(got[name], joined), name
        else:  # the same numbers added in another order, and rounded
            far = (got[name].double() - joined.double()).norm() / joined.double().norm()
            assert float(far) <= 2.0**-9, (name, float(far))  # two roundings of 2^-8 / sqrt(3) at most each, and few differ
    want = attention64(q[:, :1], k[:, :1], v[:, :1], o, o, causal, None, d_out[:, :1])
    for name in got:
        check(got[name][:, :1], want[name], name)


def test_one_sequence_without_offsets(dev):
    import torch

    q, k, v, d_out = inputs(dev, 150, 150, 4, 2, 64)
    a = gradients(q, k, v, d_out)
    b = gradients(q, k, v, d_out, index([0, 150], dev))
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_rows_of_no_sequence_are_zero(dev):
    """Rows before the first sequence and behind the last one, of results and
    gradients, and what the sequences get is what they get alone."""
    import torch

    q, k, v, d_out = inputs(dev, 100, 100, 4, 2, 64)
    for t in (q, k, v, d_out):
        t[:7] = float("nan")
        t[80:] = float("nan")
    got = gradients(q, k, v, d_out, index([7, 30, 80], dev))
    alone = gradients(q[7:80], k[7:80], v[7:80], d_out[7:80], index([0, 23, 73], dev))
    for name in got:
        assert not got[name][:7].any() and not got[name][80:].any()
        assert torch.equal(got[name][7:80], alone[name]), name


def test_offsets_out_of_range_are_clamped(dev):
    import torch

    q, k, v, d_out = inputs(dev, 50, 50, 2, 2, 64)
    a = gradients(q, k, v, d_out, index([-5, 20, 1 << 30], dev))
    b = gradients(q, k, v, d_out, index([0, 20, 50], dev))
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_no_rows(dev):
    import torch

    M = pkg()
    q = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=dev)
    k = torch.randn(9, 2, 64, device=dev).to(torch.bfloat16)
    assert M.packed_attention(q, q[:, :2], q[:, :2]).shape == (0, 4, 64)
    got = gradients(q, k, k, q, index([0, 0], dev), index([0, 9], dev))
    assert got["d_k"].shape == k.shape and not got["d_k"].any() and not got["d_v"].any()
    q = torch.randn(9, 4, 64, device=dev).to(torch.bfloat16)
    got = gradients(q, k[:0], k[:0], q, index([0, 9], dev), index([0, 0], dev))
    assert not got["out"].any() and not got["d_q"].any() and got["d_k"].shape == (0, 2, 64)


def test_views_without_copies_and_with(dev):
    """Slices of one joint tensor, head-major tensors, rows at odd addresses,
    gradients that are expanded: the same bits as contiguous ones."""
    import torch

    q, k, v, d_out = inputs(dev, 90, 90, 6, 2, 64)
    o = index([0, 40, 90], dev)
    want = gradients(q, k, v, d_out, o)
    joint = torch.cat([q, k, v], 1)
    views = joint.split([6, 2, 2], 1)
    A = submodule("attention")
    assert all(A.head_rows(t)[0] is t for t in views)
    head_major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert all(A.head_rows(t)[0] is t for t in head_major)
    odd = []
    for t in (q, k, v):
        room = torch.empty(t.numel() + 1, dtype=torch.bfloat16, device=dev)[1:].view(t.shape)
        odd.append(room.copy_(t))
    wide = [torch.stack([t, t], 3)[..., 0] for t in (q, k, v)]
    for given in (views, head_major, odd, wide):
        got = gradients(*given, d_out.transpose(0, 1).contiguous().transpose(0, 1), o)
        assert all(torch.equal(got[n], want[n]) for n in got)
    ones = torch.ones(1, 1, 1, dtype=torch.bfloat16, device=dev).expand(90, 6, 64)
    a, b = gradients(q, k, v, ones, o), gradients(q, k, v, ones.contiguous(), o)
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_shared_keys_by_expansion(dev):
    """Keys expanded over heads: the gradient of the one behind them is the sum
    that grouped heads give, up to each term's own rounding."""
    import torch

    q, k, v, d_out = inputs(dev, 80, 80, 4, 1, 64)
    k, v = k.requires_grad_(), v.requires_grad_()
    out = pkg().packed_attention(q, k.expand(80, 4, 64), v.expand(80, 4, 64))
    dk, dv = torch.autograd.grad(out, [k, v], d_out)
    want = gradients(q, k, v, d_out)
    assert torch.equal(out, want["out"])
    for got, name in ((dk, "d_k"), (dv, "d_v")):
        # four terms rounded to bf16, then their sum; each at most 2^-8 of magnitudes that add up
        per_head = [gradients(q[:, h:h + 1], k, v, d_out[:, h:h + 1])[name].double().abs() for h in range(4)]
        assert bool(((got.double() - want[name].double()).abs() <= 4 * 2.0**-8 * sum(per_head) + 2.0**-8 * got.double().abs()).all())


def test_single_gradients_are_the_joint_ones(dev):
    """Each subset of wanted gradients has the bits of the joint call."""
    import torch

    q, k, v, d_out, args, want = run(dev, [100, 60], [100, 60], 4, 2, 128, True)
    A = submodule("attention")
    out, lse = A.native_packed_attention(q, k, v, *args, True, 128**-0.5, True)
    for wanted in ([1, 0, 0], [0, 1, 0], [0, 0, 1], [1, 1, 0], [0, 1, 1], [1, 0, 1]):
        grads = A.native_packed_attention_backward(q, k, v, *args, out, lse, d_out, True, 128**-0.5, [bool(w) for w in wanted])
        for g, w, name in zip(grads, wanted, ("d_q", "d_k", "d_v")):
            assert (g is not None) == bool(w)
            assert g is None or torch.equal(g, want[name]), (wanted, name)


@pytest.mark.parametrize("dim", [64, 128])
def test_gradients_of_short_sequences(dev, dim):
    """Rows of few keys have large results, whose rounding shifts a whole row's dS:
    d_q must be off by its own rounding alone.  That is at most half a step, 2^-8 of a
    step's lowest value, equally likely anywhere, so 2^-7 / sqrt(12) of the root mean
    square at most; and 5% for everything in FP32 and dS's two parts (2^-17)."""
    import torch

    lengths = torch.randint(8, 101, (30,), generator=torch.Generator().manual_seed(3)).tolist()
    offsets = offsets_of(lengths)
    q, k, v, d_out = inputs(dev, offsets[-1], offsets[-1], 8, 2, dim)
    got = gradients(q, k, v, d_out, index(offsets, dev))["d_q"].double()
    want = attention64(q, k, v, offsets, offsets, True, None, d_out)["d_q"][0]
    assert float((got - want).norm() / want.norm()) <= 1.05 * 2.0**-7 / 12**0.5


def test_gradients_against_differences(dev):
    """The slope of a weighted sum of results along random directions: bf16
    results differ by steps, so the difference is taken of the 64-bit formula,
    which the results are checked against elsewhere."""
    import torch

    q, k, v, d_out = inputs(dev, 40, 40, 4, 2, 64)
    got = gradients(q, k, v, d_out)
    g = torch.Generator().manual_seed(5)
    for name, at in (("d_q", 0), ("d_k", 1), ("d_v", 2)):
        leaves = [t.double() for t in (q, k, v)]
        way = torch.randn(leaves[at].shape, generator=g).double().to(dev)
        step = 1e-5

        def value(sign):
            moved = [t + sign * step * way if i == at else t for i, t in enumerate(leaves)]
            return float((attention64(*moved, [0, 40], [0, 40], True)["out"][0] * d_out.double()).sum())

        slope = (value(1) - value(-1)) / (2 * step)
        along = got[name].double() * way
        # each gradient off by 2^-8 twice (operand, result) and delta's share, independent signs: the sum of n
        # of them by 3 * 2^-8 * the root of the squares' sum, four deviations' worth
        assert abs(float(along.sum()) - slope) <= 12 * 2.0**-8 * float(along.norm()), name


@pytest.mark.parametrize("scale", [1e-3, 0.5, 4.0])
def test_scales(dev, scale):
    run(dev, [60, 70], [60, 70], 4, 2, 64, True, scale=scale)


def test_large_scores(dev):
    """Scores up to some hundreds: rows where one key takes everything, and maxima
    that grow from tile to tile."""
    import torch

    q, k, v, d_out = inputs(dev, 300, 300, 2, 1, 64)
    k *= torch.linspace(0.1, 12, 300, device=dev).to(torch.bfloat16)[:, None, None]
    got = gradients(q, k, v, d_out, index([0, 300], dev), causal=False)
    want = attention64(q, k, v, [0, 300], [0, 300], False, None, d_out)
    # exp2's argument reaches 2^11: its rounding is 2^-24 of that, 2^-13 of a weight, 2^5 times what FP32 counts
    for name in got:
        value, bound = want[name]
        assert float((got[name].double() - value).norm() / value.norm()) <= 2 * 2.0**-8, name
    assert bool(got["out"].isfinite().all())


def test_same_bits_every_time(dev):
    import torch

    q, k, v, d_out = inputs(dev, 700, 700, 8, 2, 128)
    o = index([0, 300, 301, 700], dev)
    first = gradients(q, k, v, d_out, o)
    for _ in range(3):
        again = gradients(q, k, v, d_out, o)
        assert all(torch.equal(first[n], again[n]) for n in first)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_infinities_reach_only_what_sees_them(dev, value, dim):
    """A NaN or infinity in one token of one sequence: the rows that do not see
    that token keep their bits, in results and gradients, and so does every
    other sequence; of the values, only the column that holds it changes."""
    import torch

    lengths = [90, 150, 40]
    o, at = offsets_of(lengths), 90 + 70
    q, k, v, d_out = inputs(dev, o[-1], o[-1], 4, 2, dim)
    clean = gradients(q, k, v, d_out, index(o, dev))
    sequence = slice(90, 240)
    other = torch.ones(o[-1], dtype=torch.bool, device=dev)
    other[sequence] = False

    def same(got, name, rows, message):
        assert torch.equal(got[name][rows], clean[name][rows]), (message, name)

    # values: rows before it do not see it
    w = v.clone()
    w[at, 1, 5] = value
    got = gradients(q, k, w, d_out, index(o, dev))
    for name in ("out", "d_q"):
        same(got, name, slice(0, at), "v")
        same(got, name, slice(240, None), "v")
    assert not got["out"][at:240, 2:, 5].isfinite().any()  # heads 2 and 3 read key head 1
    assert torch.equal(got["out"][..., :5], clean["out"][..., :5]) and torch.equal(got["out"][:, :2], clean["out"][:, :2])
    same(got, "d_v", slice(None), "v")  # P does not know of v
    same(got, "d_k", other, "v")
    # a key: only rows from it on see it
    w = k.clone()
    w[at, 1, 5] = value
    got = gradients(q, w, v, d_out, index(o, dev))
    for name in ("out", "d_q"):
        same(got, name, slice(0, at), "k")
        same(got, name, slice(240, None), "k")
    for name in ("d_k", "d_v"):
        same(got, name, other, "k")
    if value != value:
        assert got["out"][at:240, 2:].isnan().all()
    # a query: its own results, and the keys that it sees
    w = q.clone()
    w[at, 3, 5] = float("nan")
    got = gradients(w, k, v, d_out, index(o, dev))
    assert got["out"][at, 3].isnan().all() and got["d_q"][at, 3].isnan().all()
    kept = torch.ones(o[-1], 4, dtype=torch.bool, device=dev)
    kept[at, 3] = False
    for name in ("out", "d_q"):
        assert torch.equal(got[name][kept], clean[name][kept])
    for name in ("d_k", "d_v"):
        same(got, name, slice(0, 90), "q")
        same(got, name, slice(at + 1, None), "q")
        assert got[name][90:at + 1, 1].isnan().all()
    # a result's gradient: d_v of the keys that its row sees, in its column alone
    w = d_out.clone()
    w[at, 3, 5] = value
    got = gradients(q, k, v, w, index(o, dev))
    same(got, "out", slice(None), "d_out")
    assert torch.equal(got["d_q"][kept], clean["d_q"][kept])
    for name in ("d_k", "d_v"):
        same(got, name, slice(0, 90), "d_out")
        same(got, name, slice(at + 1, None), "d_out")
    rest = [c for c in range(dim) if c != 5]
    assert torch.equal(got["d_v"][..., rest], clean["d_v"][..., rest])
    assert not got["d_v"][90:at + 1, 1, 5].isfinite().any()


def test_offsets_past_32_bits(dev):
    """Rows so far apart that their places pass 2^32 bytes and elements."""
    import torch

    tokens, stride = 70_000, 1 << 16
    room = torch.empty(tokens, stride, dtype=torch.bfloat16, device=dev)
    view = room[:, :5 * 64].view(tokens, 5, 64)
    g = torch.Generator(device=dev).manual_seed(0)
    view.copy_(torch.randn(tokens, 5, 64, generator=g, device=dev))
    q, k, v = view.split([3, 1, 1], 1)
    assert submodule("attention").head_rows(q)[0] is q
    o = list(range(0, tokens, 100)) + [tokens]
    got = gradients(q, k, v, q.contiguous(), index(o, dev))
    last = slice(tokens - 100, tokens)
    want = attention64(q[last], k[last], v[last], [0, 100], [0, 100], True, None, q[last])
    for name in got:
        check(got[name][last], want[name], name)


@pytest.mark.parametrize("sequences", [61, 62, 63, 64, 65, 200])
def test_many_sequences(dev, sequences):
    """Around as many as a wavefront has lanes."""
    lengths = [1 + (7 * i) % 11 for i in range(sequences)]
    run(dev, lengths, lengths, 2, 1, 64, True)


@pytest.mark.parametrize("sequences", [4094, 4095, 4200])
def test_searched_in_several_steps(dev, sequences):
    """More sequences than 64 * 64 segments, some of them empty."""
    import torch

    lengths = torch.randint(0, 4, (sequences,), generator=torch.Generator().manual_seed(1)).tolist()
    run(dev, lengths, lengths, 2, 1, 64, True)


@pytest.mark.parametrize("lengths", [[2300, 2100], [4300, 0, 100]])
def test_long_sequences_first(dev, lengths):
    """Lengths whose tiles are taken longest first."""
    import torch

    o = offsets_of(lengths)
    q, k, v, d_out = inputs(dev, o[-1], o[-1], 2, 1, 64)
    got = gradients(q, k, v, d_out, index(o, dev))
    for a, b in zip(o[:-1], o[1:]):
        if a == b:
            continue
        alone = gradients(q[a:b], k[a:b], v[a:b], d_out[a:b])
        for name in got:
            assert torch.equal(got[name][a:b], alone[name]), name


def test_captured_and_replayed(dev):
    """A forward and backward call in one graph, replayed over new inputs and
    new offsets with eager work between, equals the eager calls."""
    import torch

    A = submodule("attention")
    q, k, v, d_out = inputs(dev, 120, 120, 4, 2, 64)
    o = index([0, 50, 120], dev)
    static = [t.clone() for t in (q, k, v, d_out, o)]

    def step():
        out, lse = A.native_packed_attention(*static[:3], static[4], None, True, 0.125, True)
        return [out, *A.native_packed_attention_backward(*static[:3], static[4], None, out, lse, static[3], True, 0.125, [True] * 3)]

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        results = step()
    for seed, offsets in ((1, [0, 50, 120]), (2, [0, 119, 120]), (3, [3, 3, 90])):
        new = inputs(dev, 120, 120, 4, 2, 64, seed)
        for s, t in zip(static, (*new, index(offsets, dev))):
            s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = gradients(*new, index(offsets, dev), scale=0.125)
        for got, name in zip(results, ("out", "d_q", "d_k", "d_v")):
            assert torch.equal(got, want[name]), (seed, name)


def test_two_streams_at_once(dev):
    import torch

    sets = [inputs(dev, 800, 800, 8, 2, 128, seed) for seed in (1, 2)]
    want = [gradients(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[] for _ in sets]
    for _ in range(3):
        for i, (s, stream) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(stream):
                got[i].append(gradients(*s))
    torch.cuda.synchronize()
    for w, all_got in zip(want, got):
        for g in all_got:
            assert all(torch.equal(g[n], w[n]) for n in w)


def test_as_a_custom_op(dev):
    """Traced, and with the registered gradient: the eager call's bits."""
    import torch

    M = pkg()
    q, k, v, d_out = inputs(dev, 60, 60, 4, 2, 64)
    want = gradients(q, k, v, d_out, index([0, 25, 60], dev))
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    o = index([0, 25, 60], dev)
    out, lse = torch.ops.glm53.packed_attention(q, k, v, o, None, True, 0.125, True)
    grads = torch.autograd.grad(out, [q, k, v], d_out)
    assert torch.equal(out, want["out"])
    assert all(torch.equal(g, want[n]) for g, n in zip(grads, ("d_q", "d_k", "d_v")))
    with torch.no_grad():
        traced = torch.compile(lambda a, b, c: M.packed_attention(a, b, c, o), backend="eager", fullgraph=True)
        assert torch.equal(traced(q, k, v), want["out"])
    torch.library.opcheck(torch.ops.glm53.packed_attention.default, (q.detach(), k.detach(), v.detach(), o, None, True, 0.125, False))


def test_refused_transforms(dev):
    import torch

    q, k, v, _ = inputs(dev, 10, 10, 2, 1, 64)
    for call in (lambda: torch.func.jvp(lambda a: pkg().packed_attention(a, k, v), (q,), (q,)),
                 lambda: torch.func.grad(lambda a: pkg().packed_attention(q, a, v).float().sum())(k)):
        with pytest.raises(RuntimeError, match="no derivative"):
            call()


def test_python_refusals(dev):
    import torch

    M = pkg()
    q, k, v, _ = inputs(dev, 10, 10, 4, 2, 64)
    o = index([0, 10], dev)
    wrong = [
        (q.float(), k, v), (q, k.half(), v), (q[0], k, v), (q, k[:, :1], v), (q, k, v[..., :32]), (q[:, :3], k, v),
        (q, k[:9], v[:9]), (q, k, v, o, index([0, 5, 10], dev)), (q, k, v, None, o), (q, k, v, o.long()),
        (q, k, v, o[:1]), (q, k, v, o[None]), (q[..., :60].contiguous(), k[..., :60].contiguous(), v[..., :60].contiguous()),
        (torch.zeros(4, 2, 264, dtype=torch.bfloat16, device=dev),) * 3, (q, k.cpu(), v), (q, k, v, o.cpu()),
    ]
    for args in wrong:
        with pytest.raises((ValueError, RuntimeError)):
            M.packed_attention(*args)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            M.packed_attention(q, k, v, scale=scale)
