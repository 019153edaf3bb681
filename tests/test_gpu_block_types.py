"""GPU tests of runs of blocks whose feed-forwards return FP32."""

from __future__ import annotations

import pytest

from conftest import pkg

pytestmark = pytest.mark.gpu


def _blocks(dev, dtype):
    import torch

    M = pkg()

    class Wide(torch.nn.Module):
        """A feed-forward of bfloat16 input that returns another type."""

        def __init__(self):
            super().__init__()
            self.mlp = M.GatedMLP(64, 32, limit=4.0, device=dev)

        def forward(self, x):
            assert x.dtype == torch.bfloat16
            return self.mlp(x).to(dtype)

    torch.manual_seed(0)
    return [M.FeedForwardBlock(Wide(), 64, device=dev) for _ in range(3)], torch.ones(64, device=dev, dtype=torch.bfloat16)


@pytest.mark.parametrize("residual", ["bfloat16", "float32"])
def test_feed_forwards_that_return_fp32(dev, residual):
    """Each block's input is bfloat16, whatever the block before returned; the
    run is its blocks alone, and has the gradients of the FP32 values rounded."""
    import torch

    M = pkg()
    x = torch.randn(9, 64, device=dev).to(getattr(torch, residual))
    blocks, final = _blocks(dev, torch.float32)
    same, _ = _blocks(dev, torch.bfloat16)  # the same values, returned in bfloat16
    r, y = M.run_blocks(blocks, x, final)
    wr, wy = M.run_blocks(same, x, final)
    assert r.dtype == x.dtype and torch.equal(r, wr)
    assert torch.equal(y.to(torch.bfloat16), wy)
    given = torch.randn(9, 64, device=dev).to(x.dtype)
    got = torch.autograd.grad(r, blocks[0].mlp.mlp.gate_proj.weight, given)[0]
    want = torch.autograd.grad(wr, same[0].mlp.mlp.gate_proj.weight, given)[0]
    # FP32 block outputs keep their gradients in FP32 on the way: 6 roundings of bf16 fewer or more
    assert float((got.double() - want.double()).norm()) <= 6 * 2.0**-8 * float(want.double().norm())
