"""GPU tests of the dense block's products at sizes whose grids or joins pass
2^32 threads: the rows of a small call, repeated."""

from __future__ import annotations

import pytest

from conftest import pkg

pytestmark = pytest.mark.gpu


def _repeats(y, part):
    """Whether every run of part's rows in y is `part`, looked at in pieces."""
    import torch

    rows = part.shape[0]
    step = (1 << 27) // part.numel() * rows
    pieces = (y[at:at + step].view(-1, *part.shape) for at in range(0, y.shape[0], step))
    return all(bool((p == part).all()) for p in pieces)


@pytest.fixture(autouse=True)
def _free(dev):
    import torch

    yield
    torch.cuda.empty_cache()


def test_4_bit_products_of_2_to_the_34_results(dev):
    """Results beyond the grid of the pass that joins partial results, which a
    product in one part does not have."""
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    rows, n, k, base = 1 << 22, 4096, 32, 256
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.rand(n, 1, generator=g, device="cuda").to(torch.bfloat16)
    x = torch.randn(base, k, generator=g, device="cuda").to(torch.bfloat16)
    y = pkg().int4_linear(x.repeat(rows // base, 1), codes, scales)
    assert y.shape == (rows, n)
    assert _repeats(y, pkg().int4_linear(x, codes, scales))


def test_gated_mlp_over_almost_2_to_the_31_rows(dev):
    """The most rows: tiles of more than 2^32 threads, in several launches."""
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    rows, width, base = (1 << 31) - 64, 8, 64
    x, gate, up, down = (torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)
                         for s in ((base, width), (width, width), (width, width), (width, width)))
    y = pkg().gated_mlp(x.repeat(rows // base, 1), gate, up, down, 2.0)
    assert y.shape == (rows, width)
    assert _repeats(y, pkg().gated_mlp(x, gate, up, down, 2.0))
