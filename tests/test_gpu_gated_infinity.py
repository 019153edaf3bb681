"""GPU tests of infinite weights in the gated MLP over few rows, which
multiply h in two bf16 parts: infinities of the formula stay infinities."""

from __future__ import annotations

import pytest

from conftest import pkg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 2, 16, 17, 32, 33, 100])
@pytest.mark.parametrize("value", ["inf", "-inf", "nan"])
def test_an_infinite_weight_is_its_column_s_own_affair(dev, rows, value):
    """y = h Wd^T with one infinite weight in Wd: h times infinity in its column
    of y, all others as they were."""
    import torch

    M = pkg()
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)

    x, gate, up, down = normal(rows, 256), normal(128, 256, std=0.1), normal(128, 256, std=0.1), normal(64, 128)
    down = torch.cat([down, down, down, down])
    clean = M.gated_mlp(x, gate, up, down, 3.0)
    bad = down.clone()
    bad[7, 5] = float(value)
    y = M.gated_mlp(x, gate, up, bad, 3.0)
    G, U = x[:, None, :].double() @ gate.t().double(), x[:, None, :].double() @ up.t().double()
    h = (G.clamp(max=3.0) * torch.sigmoid(G.clamp(max=3.0)) * U.clamp(-3.0, 3.0))[:, 0, 5]
    assert torch.equal(y[:, 7].double(), h * float(value)) or (value == "nan" and y[:, 7].isnan().all())
    keep = [n for n in range(256) if n != 7]
    assert torch.equal(y[:, keep], clean[:, keep])
