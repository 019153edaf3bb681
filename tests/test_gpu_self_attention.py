"""GPU tests of attention as it is used: in blocks with norms and
feed-forwards, trained, and served chunk by chunk and token by token over a
cache."""

from __future__ import annotations

import pytest

from conftest import pkg

pytestmark = pytest.mark.gpu


def index(values, dev):
    import torch

    return torch.tensor(values, dtype=torch.int32, device=dev)


def model(dev, hidden=256, heads=8, kv_heads=2, dim=64, layers=2):
    """Blocks of attention and of a gated MLP in turn."""
    import torch

    M = pkg()
    torch.manual_seed(0)
    blocks = []
    for _ in range(layers):
        blocks.append(M.FeedForwardBlock(M.SelfAttention(hidden, heads, kv_heads, dim, device=dev), hidden, device=dev))
        blocks.append(M.FeedForwardBlock(M.GatedMLP(hidden, 128, 4.0, device=dev), hidden, residual_scale=0.5, device=dev))
    return torch.nn.ModuleList(blocks), torch.ones(hidden, device=dev, dtype=torch.bfloat16)


def reference(blocks, x, final, offsets, given=None):
    """The same in 64 bits, sequence by sequence, with torch's own gradients."""
    import torch

    leaves = {n: p.detach().double().requires_grad_() for n, p in blocks.named_parameters()}
    x0 = x.detach().double().requires_grad_()

    def norm(v, w, eps):
        return v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * w

    r = x0
    for i, b in enumerate(blocks):
        w = {n.split(".", 1)[1]: p for n, p in leaves.items() if n.startswith(f"{i}.")}
        h = norm(r, w["norm_weight"], b.eps)
        if hasattr(b.mlp, "qkv_proj"):
            a = b.mlp
            rows = (h @ w["mlp.qkv_proj.weight"].t()).view(-1, a.heads + 2 * a.kv_heads, a.head_dim)
            q, k, v = rows.split([a.heads, a.kv_heads, a.kv_heads], 1)
            k, v = (t.repeat_interleave(a.heads // a.kv_heads, 1) for t in (k, v))
            parts = []
            for s, e in zip(offsets[:-1], offsets[1:]):
                qq, kk, vv = (t[s:e].transpose(0, 1) for t in (q, k, v))
                seen = torch.ones(e - s, e - s, dtype=torch.bool, device=x.device).tril()
                p = (qq @ kk.transpose(1, 2) * a.head_dim**-0.5).masked_fill(~seen, -float("inf")).softmax(-1)
                parts.append((p @ vv).transpose(0, 1))
            o = torch.cat(parts).reshape(len(h), -1) @ w["mlp.o_proj.weight"].t()
        else:
            g, u = (h @ w["mlp.gate_proj.weight"].t()).clamp(max=4.0), (h @ w["mlp.up_proj.weight"].t()).clamp(-4.0, 4.0)
            o = (g * torch.sigmoid(g) * u) @ w["mlp.down_proj.weight"].t()
        r = r + b.residual_scale * norm(o, w["post_weight"], b.eps)
    y = norm(r, final.double(), blocks[-1].eps)
    if given is None:
        return r, y
    grads = torch.autograd.grad([r, y], [x0, *leaves.values()], [g.double() for g in given])
    return r, y, dict(zip(["x", *leaves], grads))


def far(got, want):
    return float((got.detach().double() - want.detach()).norm() / want.detach().norm())


def test_trained_blocks(dev):
    """A packed batch through attention and MLP blocks on an fp32 residual
    stream: outputs and every gradient.  bf16 roundings on the way: of normed, joint
    projection, P, attention and projection in an attention block (5), of
    normed, h and out in an MLP's (3), twice as many in their backward; each 2^-8 / sqrt(3)
    of a term or less, so the 3 * 16 of two pairs make less than sqrt(48) 2^-8 /
    sqrt(3) = 4 * 2^-8 of a result whose terms do not cancel; twice that for what does."""
    import torch

    M = pkg()
    blocks, final = model(dev)
    offsets = [0, 70, 71, 150]
    x = torch.randn(150, 256, device=dev).requires_grad_()
    given = [torch.randn(150, 256, device=dev), torch.randn(150, 256, device=dev).to(torch.bfloat16)]
    batch = M.AttentionBatch(offsets=index(offsets, dev))
    r, y = M.run_blocks(blocks, x, final, batch)
    names = ["x", *(n for n, _ in blocks.named_parameters())]
    grads = dict(zip(names, torch.autograd.grad([r, y], [x, *blocks.parameters()], given)))
    wr, wy, wg = reference(blocks, x, final, offsets, given)
    assert far(r, wr) <= 8 * 2.0**-8 and far(y, wy) <= 8 * 2.0**-8
    for n in names:
        assert far(grads[n], wg[n]) <= 8 * 2.0**-8, (n, far(grads[n], wg[n]))


def test_batched_and_single_sequences(dev):
    """[sequences, length, hidden] is the packed batch of equal lengths, and
    [length, hidden] one sequence."""
    import torch

    M = pkg()
    torch.manual_seed(0)
    a = M.SelfAttention(128, 4, 2, 64, device=dev)
    x = torch.randn(3, 40, 128, device=dev).to(torch.bfloat16)
    with torch.no_grad():
        y = a(x)
        packed = a(x.view(120, 128), M.AttentionBatch(offsets=index([0, 40, 80, 120], dev)))
        assert torch.equal(y.view(120, 128), packed)
        # the projections of 40 rows may be another library kernel's than those of 120
        for i in range(3):
            assert far(a(x[i]), y[i].double()) <= 2.0**-7
        assert a(x[:, :0]).shape == (3, 0, 128) and a(x[:0]).shape == (0, 40, 128)
    both = M.SelfAttention(128, 4, 2, 64, causal=False, scale=0.1, device=dev)
    assert both(x).isfinite().all()


def test_optimiser_steps_run(dev):
    import torch

    M = pkg()
    blocks, final = model(dev)
    opt = torch.optim.SGD(blocks.parameters(), lr=1e-2)
    before = [p.detach().clone() for p in blocks.parameters()]
    x = torch.randn(2, 30, 256, device=dev).to(torch.bfloat16)
    for _ in range(2):
        opt.zero_grad()
        _, y = M.run_blocks(blocks, x, final)
        y.float().square().mean().backward()
        assert all(p.grad is not None and p.grad.isfinite().all() for p in blocks.parameters())
        opt.step()
    assert any(not torch.equal(a, b) for a, b in zip(before, blocks.parameters()))


def tables(dev, sequences, pages_each):
    import torch

    order = torch.randperm(sequences * pages_each, generator=torch.Generator().manual_seed(1))
    return order.view(sequences, pages_each).to(torch.int32).to(dev)


@pytest.mark.parametrize("quantised", [False, True])
@pytest.mark.parametrize("served", [False, True])
def test_served_in_chunks_and_tokens(dev, quantised, served):
    """Prompts in a first chunk, a second chunk over the cache, then tokens one
    by one: each step's rows are those of the whole sequences at once.  In bf16 by
    the roundings of test_trained_blocks' forward (24 of 2^-8 / sqrt(3): 2.9 *
    2^-8, twice that); an E4M3 cache adds 2^-4 / sqrt(3) of each key and value,
    0.036 of a result at each of two layers, and as much again through the scores."""
    import torch

    M = pkg()
    blocks, final = model(dev)
    if served:
        for b in blocks:
            b.mlp = b.mlp.to_int4(group_size=32)
    attentions = [b.mlp for b in blocks if hasattr(b.mlp, "cache")]
    first, second, steps = [50, 7, 64], [20, 33, 1], 5
    total = [a + b + steps for a, b in zip(first, second)]
    x = [torch.randn(n, 256, device=dev).to(torch.bfloat16) for n in total]
    for a in attentions:
        a.cache = M.KVCache(3 * 8, 16, a.kv_heads, a.head_dim, quantised=quantised, device=dev)
    table = tables(dev, 3, 8)

    def offsets(lengths):
        got = [0]
        for n in lengths:
            got.append(got[-1] + n)
        return got

    def rows(start, lengths):
        return torch.cat([t[s:s + n] for t, s, n in zip(x, start, lengths)])

    with torch.no_grad():
        whole = M.run_blocks(blocks, torch.cat(x), final, M.AttentionBatch(offsets=index(offsets(total), dev)))[1]
        whole = whole.split(total)
        limit = 6 * 2.0**-8 if not quantised else 6 * 2.0**-8 + 4 * 2.0**-4 / 3**0.5

        def near(got, start, lengths):
            want = torch.cat([t[s:s + n] for t, s, n in zip(whole, start, lengths)])
            assert far(got, want.double()) <= limit, far(got, want.double())

        zero = [0, 0, 0]
        batch = M.AttentionBatch(offsets=index(offsets(first), dev), page_table=table, lengths=index(zero, dev))
        near(M.run_blocks(blocks, rows(zero, first), final, batch)[1], zero, first)
        now = [a + b for a, b in zip(first, second)]
        batch = M.AttentionBatch(offsets=index(offsets(second), dev), page_table=table, lengths=index(first, dev),
                                 key_offsets=index(offsets(now), dev), keys=sum(now))
        near(M.run_blocks(blocks, rows(first, second), final, batch)[1], first, second)
        for _ in range(steps):
            batch = M.AttentionBatch(page_table=table, lengths=index(now, dev))
            near(M.run_blocks(blocks, rows(now, [1, 1, 1]), final, batch)[1], now, [1, 1, 1])
            now = [n + 1 for n in now]


def test_captured_decode_steps(dev):
    """A whole decode step of 4-bit blocks in one graph, replayed as the
    sequences grow: the eager steps' bits."""
    import torch

    M = pkg()
    blocks, final = model(dev)
    for b in blocks:
        b.mlp = b.mlp.to_int4(group_size=32)
    attentions = [b.mlp for b in blocks if hasattr(b.mlp, "cache")]

    def caches():
        for a in attentions:
            a.cache = M.KVCache(2 * 8, 16, a.kv_heads, a.head_dim, quantised=True, device=dev)
        return [a.cache for a in attentions]

    table = tables(dev, 2, 8)
    x = torch.zeros(2, 256, device=dev, dtype=torch.bfloat16)
    batch = M.AttentionBatch(page_table=table, lengths=index([0, 3], dev))
    own = caches()
    stream = torch.cuda.Stream()
    with torch.no_grad():
        with torch.cuda.stream(stream):
            M.run_blocks(blocks, x, final, batch)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = M.run_blocks(blocks, x, final, batch)[1]
        other = caches()
        for a, b in zip(other, own):
            for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
                getattr(a, name).copy_(getattr(b, name))
        for n in range(12):
            new = torch.randn(2, 256, device=dev).to(torch.bfloat16)
            x.copy_(new)
            batch.lengths.copy_(index([n, 3 + 2 * n], dev))
            batch.after.copy_(index([n + 1, 4 + 2 * n], dev))
            graph.replay()
            torch.cuda.synchronize()
            eager = M.run_blocks(blocks, new, final, M.AttentionBatch(page_table=table, lengths=index([n, 3 + 2 * n], dev)))[1]
            assert torch.equal(out, eager), n


def test_refusals(dev):
    import torch

    M = pkg()
    a = M.SelfAttention(128, 4, 2, 64, device=dev)
    x = torch.randn(2, 128, device=dev).to(torch.bfloat16)
    batch = M.AttentionBatch(page_table=index([[0], [1]], dev), lengths=index([0, 0], dev))
    with pytest.raises(RuntimeError, match="needs a cache"):
        a(x, batch)
    both = M.SelfAttention(128, 4, 2, 64, causal=False, device=dev)
    both.cache = M.KVCache(2, 16, 2, 64, device=dev)
    with pytest.raises(RuntimeError, match="causal"):
        both(x, batch)
    # a feed-forward without attention does not see the batch
    block = M.FeedForwardBlock(M.GatedMLP(128, 64, device=dev), 128, device=dev)
    with torch.no_grad():
        assert torch.equal(M.run_blocks([block], x, None, batch)[0], M.run_blocks([block], x)[0])
