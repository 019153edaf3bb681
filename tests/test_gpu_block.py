"""GPU tests of feed-forward blocks as they are used: norms, gated MLP and
4-bit linears together, in training and served, and around the FP8 layers."""

from __future__ import annotations

import pytest

from conftest import pkg, submodule

pytestmark = pytest.mark.gpu


def _blocks(dev, hidden=256, inter=128, count=3, dtype=None):
    import torch

    M = pkg()
    torch.manual_seed(0)
    blocks = []
    for _ in range(count):
        b = M.FeedForwardBlock(M.GatedMLP(hidden, inter, limit=4.0, device=dev), hidden, gate=True, residual_scale=0.5,
                               device=dev, dtype=dtype or torch.bfloat16)
        with torch.no_grad():
            for w in (b.norm_weight, b.post_weight, b.gate):
                w.mul_(1 + 0.2 * torch.randn_like(w))
        blocks.append(b)
    return torch.nn.ModuleList(blocks), torch.ones(hidden, device=dev, dtype=dtype or torch.bfloat16)


def _reference(blocks, residual, final, given):
    """The same blocks in 64 bits with torch's own gradients."""
    import torch

    leaves = {n: p.detach().double().requires_grad_() for n, p in blocks.named_parameters()}
    x0 = residual.detach().double().requires_grad_()

    def norm(v, w, eps):
        return v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * w

    x = x0
    for i, b in enumerate(blocks):
        w = {n.split(".", 1)[1]: p for n, p in leaves.items() if n.startswith(f"{i}.")}
        h = norm(x, w["norm_weight"], b.eps)
        g = (h @ w["mlp.gate_proj.weight"].t()).clamp(max=4.0)
        u = (h @ w["mlp.up_proj.weight"].t()).clamp(-4.0, 4.0)
        o = (g * torch.sigmoid(g) * u) @ w["mlp.down_proj.weight"].t()
        x = x + b.residual_scale * w["gate"] * norm(o, w["post_weight"], b.eps)
    y = norm(x, final.double(), blocks[-1].eps)
    grads = torch.autograd.grad([x, y], [x0, *leaves.values()], [g.double() for g in given])
    return x, y, dict(zip(["residual", *leaves], grads))


def _far(got, want):
    return float((got.detach().double() - want.detach()).norm() / want.detach().norm())


def test_run_of_blocks_in_training(dev):
    """Three blocks on an fp32 residual stream: outputs and every gradient.
    bf16 roundings on the way: of normed, h and out in each block, twice as
    many in its backward; each is 2^-8 / sqrt(3) of a term or less, and the 9
    of a block's forward and backward over three blocks make less than
    sqrt(27) 2^-8 / sqrt(3) = 3 2^-8 of a result whose terms do not cancel;
    twice that for what does."""
    import torch

    blocks, final = _blocks(dev)
    x = torch.randn(4, 37, 256, device=dev).requires_grad_()
    given = [torch.randn(4, 37, 256, device=dev), torch.randn(4, 37, 256, device=dev).to(torch.bfloat16)]
    r, y = pkg().run_blocks(blocks, x, final)
    assert r.dtype == torch.float32 and y.dtype == torch.bfloat16
    names = ["residual", *(n for n, _ in blocks.named_parameters())]
    grads = torch.autograd.grad([r, y], [x, *blocks.parameters()], given)
    wr, wy, wg = _reference(blocks, x, final, given)
    assert _far(r, wr) <= 6 * 2.0**-8 and _far(y, wy) <= 6 * 2.0**-8
    for n, g in zip(names, grads):
        assert _far(g, wg[n]) <= 6 * 2.0**-8, (n, _far(g, wg[n]))


def test_blocks_joined_equal_blocks_alone(dev):
    """A norm made by the pass before is the norm made alone, up to the
    rounding of a bf16 residual; on an fp32 stream bit for bit up to FP32's."""
    import torch

    blocks, final = _blocks(dev)
    x = torch.randn(50, 256, device=dev)
    with torch.no_grad():
        r, y = pkg().run_blocks(blocks, x, final)
        alone = x
        for b in blocks:
            alone, none = b(alone)
            assert none is None
        assert torch.equal(r, alone)
        assert torch.equal(y, pkg().rms_norm(alone, final, blocks[-1].eps, dtype=torch.bfloat16))


def test_optimiser_steps_run(dev):
    import torch

    blocks, final = _blocks(dev)
    before = [p.detach().clone() for p in blocks.parameters()]
    opt = torch.optim.SGD(blocks.parameters(), lr=1e-2)
    x = torch.randn(2, 20, 256, device=dev).to(torch.bfloat16)
    for _ in range(2):
        opt.zero_grad()
        _, y = pkg().run_blocks(blocks, x, final)
        y.float().square().mean().backward()
        assert all(p.grad is not None and p.grad.isfinite().all() for p in blocks.parameters())
        opt.step()
    assert any(not torch.equal(a, b) for a, b in zip(before, blocks.parameters()))


@pytest.mark.parametrize("rows", [1, 5, 40])
def test_served_in_four_bits(dev, rows):
    """The trained blocks with their MLPs in 4 bits, eager and replayed from a
    captured graph: each step is the operators' own composition."""
    import torch

    M = pkg()
    blocks, final = _blocks(dev)
    for b in blocks:
        b.mlp = b.mlp.to_int4(group_size=64)
    x = torch.randn(rows, 256, device=dev).to(torch.bfloat16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.no_grad():
        with torch.cuda.stream(s):
            M.run_blocks(blocks, x, final)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                got = M.run_blocks(blocks, x, final)
        torch.cuda.current_stream().wait_stream(s)
        for k in range(3):
            x.copy_(torch.randn(rows, 256, device=dev))
            graph.replay()
            torch.cuda.synchronize()
            want = M.run_blocks(blocks, x, final)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        r, n = x, None
        for i, b in enumerate(blocks):
            n = M.rms_norm(r, b.norm_weight, b.eps) if n is None else n
            m = b.mlp
            j = M.int4_linear(n, m.gate_up_proj.weight, m.gate_up_proj.scales, m.gate_up_proj.offsets)
            h = M.swiglu(j[:, :128], j[:, 128:], 4.0)
            o = M.int4_linear(h, m.down_proj.weight, m.down_proj.scales, m.down_proj.offsets)
            w = blocks[i + 1].norm_weight if i + 1 < len(blocks) else final
            r, n = M.residual_norm(r, o, post_weight=b.post_weight, gate=b.gate, scale=b.residual_scale, next_weight=w,
                                   eps=b.eps)
        assert torch.equal(r, want[0]) and torch.equal(n, want[1])


@pytest.mark.parametrize("tokens", [1, 40])
def test_around_the_fp8_moe(dev, tokens):
    """A block around a SortedGroupedFP8MoE is rms_norm, the layer, residual_norm."""
    import torch

    M = pkg()
    syn = submodule("synthetic")
    cfg = syn.layer_config(hidden=1024, intermediate=512, experts=32, top_k=8, limit=10.0)
    bank, shared, gate = syn.synth_layer(cfg, seed=3, device=dev)
    moe = M.SortedGroupedFP8MoE(bank, cfg, gate, shared)
    block = M.FeedForwardBlock(moe, 1024, device=dev, residual_scale=0.5)
    x = torch.randn(1, tokens, 1024, device=dev).to(torch.bfloat16)
    token_gate = torch.rand(1, tokens, 1, device=dev)
    with torch.no_grad():
        r, n = block(x, next_weight=block.norm_weight, gate=token_gate)
        out = moe(M.rms_norm(x, block.norm_weight, 1e-6))
        wr, wn = M.residual_norm(x, out, post_weight=block.post_weight, gate=token_gate, scale=0.5,
                                 next_weight=block.norm_weight)
    assert torch.equal(r, wr) and torch.equal(n, wn)


def test_training_step_in_a_captured_graph(dev):
    """Forward and backward captured once no eager graph of the leaves lives,
    replayed with new values between eager work."""
    import torch

    blocks, final = _blocks(dev, count=2)
    x = torch.randn(24, 256, device=dev)
    dy = torch.randn(24, 256, device=dev).to(torch.bfloat16)
    params = list(blocks.parameters())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())

    def step():
        _, y = pkg().run_blocks(blocks, x, final)
        return torch.autograd.grad(y, params, dy)

    with torch.cuda.stream(s):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = step()
    torch.cuda.current_stream().wait_stream(s)
    for k in range(3):
        x.copy_(torch.randn(24, 256, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step())), k


def test_refusals(dev):
    M = pkg()
    blocks, final = _blocks(dev, count=2)
    blocks[1].eps = 1e-3
    import torch

    with pytest.raises(ValueError):
        M.run_blocks(blocks, torch.zeros(2, 256, device=dev))
    with pytest.raises(ValueError):
        M.run_blocks([], torch.zeros(2, 256, device=dev))
