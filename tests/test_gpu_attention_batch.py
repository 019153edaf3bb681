"""GPU tests of SelfAttention over a cache as a serving loop uses it: a batch
kept over steps, idle slots, prompts behind cached tokens."""

from __future__ import annotations

import pytest

from conftest import pkg
from test_gpu_self_attention import index, model, tables

pytestmark = pytest.mark.gpu


def cached_blocks(dev, quantised=False, pages=16):
    """Two layers of attention and MLPs, and a function that gives them empty caches."""
    blocks, final = model(dev)

    def fresh():
        for b in blocks:
            if hasattr(b.mlp, "cache"):
                b.mlp.cache = pkg().KVCache(pages, 16, b.mlp.kv_heads, b.mlp.head_dim, quantised=quantised, device=dev)

    return blocks, final, fresh


def rows(dev, n, seed=0):
    import torch

    return torch.randn(n, 256, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(dev)


@pytest.mark.parametrize("through", ["run_blocks", "module"])
def test_a_batch_kept_over_steps(dev, through):
    """Lengths that grow in place: each step's bits are those of a batch made for it."""
    import torch

    M = pkg()
    blocks, final, fresh = cached_blocks(dev)
    table = tables(dev, 2, 8)

    def step(x, batch):
        if through == "run_blocks":
            return M.run_blocks(blocks, x, final, batch)[1]
        return blocks[0].mlp(x, batch)

    with torch.no_grad():
        got = {}
        for kept in (True, False):
            fresh()
            batch = M.AttentionBatch(page_table=table, lengths=index([0, 5], dev))
            got[kept] = []
            for n in range(20):
                if not kept:
                    batch = M.AttentionBatch(page_table=table, lengths=index([n, 5 + n], dev))
                got[kept].append(step(rows(dev, 2, n), batch))
                batch.lengths += 1
        for a, b in zip(got[True], got[False]):
            assert torch.equal(a, b)


def test_a_captured_step_follows_the_lengths(dev):
    """Without an `after` of its own, and with the lengths changed alone."""
    import torch

    M = pkg()
    blocks, final, fresh = cached_blocks(dev)
    table = tables(dev, 2, 8)
    x, lengths = rows(dev, 2), index([0, 3], dev)
    batch = M.AttentionBatch(page_table=table, lengths=lengths)
    with torch.no_grad():
        want = []
        fresh()
        for n in range(10):
            want.append(M.run_blocks(blocks, rows(dev, 2, n), final, M.AttentionBatch(page_table=table, lengths=index([n, 3 + n], dev)))[1])
        fresh()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            M.run_blocks(blocks, x, final, batch)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = M.run_blocks(blocks, x, final, batch)[1]
        for n in range(10):
            x.copy_(rows(dev, 2, n))
            lengths.copy_(index([n, 3 + n], dev))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[n]), n


def test_a_compiled_step(dev):
    import torch

    M = pkg()
    blocks, final, fresh = cached_blocks(dev)
    fresh()
    batch = M.AttentionBatch(page_table=tables(dev, 2, 8), lengths=index([0, 3], dev))
    with torch.no_grad():
        step = torch.compile(lambda x: M.run_blocks(blocks, x, final, batch)[1], backend="eager")
        for n in range(3):
            assert torch.equal(step(rows(dev, 2, n)), M.run_blocks(blocks, rows(dev, 2, n), final, batch)[1])
            batch.lengths += 1


@pytest.mark.parametrize("quantised", [False, True])
def test_idle_slots(dev, quantised):
    """A slot without tokens and pages: attention gives it 0, the blocks a finite row, the
    other slots their own bits; one whose sequence has lost its page is NaN."""
    import torch

    M = pkg()
    blocks, final, fresh = cached_blocks(dev, quantised, pages=17)
    table = tables(dev, 2, 8)
    idle = torch.cat([table[:1], torch.full((1, 8), -1, dtype=torch.int32, device=dev), table[1:]])
    x = rows(dev, 3)
    with torch.no_grad():
        fresh()
        batch = M.AttentionBatch(page_table=idle, lengths=index([0, 0, 5], dev))
        for n in range(3):
            got = M.run_blocks(blocks, x, final, batch)[1]
            assert bool(got.isfinite().all())
            batch.lengths += index([1, 0, 1], dev)
        assert not bool(blocks[0].mlp(x, batch)[1].any())
        # the same steps with a page for the idle slot: its neighbours' rows
        fresh()
        spare = M.AttentionBatch(page_table=idle.masked_fill(idle < 0, 16), lengths=index([0, 0, 5], dev))
        for n in range(3):
            want = M.run_blocks(blocks, x, final, spare)[1]
            spare.lengths += index([1, 0, 1], dev)
        assert torch.equal(got[[0, 2]], want[[0, 2]])
        lost = M.AttentionBatch(page_table=idle, lengths=index([3, 7, 8], dev))
        got = M.run_blocks(blocks, x, final, lost)[1]
        assert bool(got[1].isnan().all()) and bool(got[[0, 2]].isfinite().all())


@pytest.mark.parametrize("through", ["run_blocks", "module"])
def test_prompts_behind_cached_tokens_need_key_offsets(dev, through):
    """Without them a step whose sequences hold tokens, which its rows would leave out, is NaN,
    captured and replayed too; over empty sequences it has the bits of a step without a cache."""
    import torch

    M = pkg()
    blocks, final, fresh = cached_blocks(dev)
    x, offsets, lengths = rows(dev, 60), index([0, 20, 35, 58], dev), index([0, 0, 0], dev)
    batch = M.AttentionBatch(offsets, tables(dev, 3, 5), lengths)

    def step(batch):
        return M.run_blocks(blocks, x, final, batch)[1] if through == "run_blocks" else blocks[0].mlp(x, batch)

    with torch.no_grad():
        fresh()
        want = step(M.AttentionBatch(offsets))
        assert torch.equal(step(batch), want)
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            step(batch)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(batch)
        for values in ([0, 0, 0], [0, 12, 0], [3, 3, 3], [0, 0, 0]):
            lengths.copy_(index(values, dev))
            graph.replay()
            torch.cuda.synchronize()
            for got in (out, step(batch)):
                if any(values):
                    assert bool(got[:58].isnan().all())
                else:
                    assert torch.equal(got, want)


def test_no_gradient_through_a_cache(dev):
    """Results over what a cache holds raise in a backward pass, instead of gradients that lack
    what went through it; a prompt's own rows have theirs."""
    import torch

    M = pkg()
    a = M.SelfAttention(256, 8, 2, 64, device=dev)
    a.cache = M.KVCache(16, 16, 2, 64, device=dev)
    table, x, offsets = tables(dev, 2, 8), rows(dev, 20), index([0, 10, 20], dev)
    y = a(x, M.AttentionBatch(offsets, table, index([0, 0], dev)))
    got = torch.autograd.grad(y.float().square().sum(), list(a.parameters()))
    y = a(x, M.AttentionBatch(offsets))
    want = torch.autograd.grad(y.float().square().sum(), list(a.parameters()))
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    chunk = M.AttentionBatch(offsets, table, index([10, 10], dev), index([0, 20, 40], dev), 40)
    y = a(x, chunk)
    with torch.no_grad():
        assert torch.equal(y, a(x, chunk))
    with pytest.raises(RuntimeError, match="no gradient"):
        y.float().sum().backward()
    y = a(x[:2], M.AttentionBatch(page_table=table, lengths=index([20, 20], dev)))
    with pytest.raises(RuntimeError, match="autograd"):
        y.float().sum().backward()
    assert all(p.grad is None or p is a.o_proj.weight for p in a.parameters())
    for p in a.parameters():  # served with frozen weights: nothing asks for one
        p.requires_grad_(False)
    assert not a(x, chunk).requires_grad
