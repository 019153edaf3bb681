"""GPU tests that 4-bit products multiply by the weights that codes, scales and
offsets define, whatever the number of rows.

Tolerances: no weight is rounded, so an FP32 sum of K products is off by at
most (K + 32) 2^-24 of the sum of the magnitudes that the kernels add, |x|
(scale (128 + q) + |offset| + 128 scale) with q up to 15; the result is rounded
once, half a step of bf16 (2^-8).  Those are worst cases, which grow with K^2:
the additions' errors, of either sign and at most 2^-24 of the magnitudes each,
have an rms of sqrt(K + 32) 2^-24 of them, and the result's rounding one of at
most 2^-8 of the result's; the rms of a whole result is held to that too."""

from __future__ import annotations

import pytest

from conftest import pkg

pytestmark = pytest.mark.gpu

STEP, HALF = 2.0**-24, 2.0**-8
ROWS = [1, 16, 17, 32, 33, 64, 100, 128, 129, 200, 300, 700]


def _problem(rows, n, k, group, offset, f32=False, seed=0):
    """Weights of scale 0.0013 or so around `offset` (None: -8 scales), and
    rows of x whose sum over each group is near zero, so that the offsets
    cancel and the codes are what is left."""
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = torch.float32 if f32 else torch.bfloat16
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = ((torch.rand(n, k // group, generator=g, device="cuda") + 0.5) * 0.0013).to(t)
    off = None
    if offset is not None:
        off = (offset * (1 + 0.1 * torch.randn(n, k // group, generator=g, device="cuda"))).to(t)
    half = torch.randn(rows, k // 2, generator=g, device="cuda").to(torch.bfloat16)
    return torch.stack([half, -half], 2).view(rows, k), codes, scales, off


def _exact(problem):
    """The product in 64 bits and the magnitudes that its FP32 sums add."""
    import torch

    x, codes, scales, off = problem
    n, k = codes.shape[0], 2 * codes.shape[1]
    q = torch.stack([codes & 15, codes >> 4], 2).view(n, k).double()
    s = scales.double().repeat_interleave(k // scales.shape[1], 1)
    o = -8 * s if off is None else off.double().repeat_interleave(k // scales.shape[1], 1)
    v = x.double()
    return v @ (s * q + o).t(), v.abs() @ (s * 271 + o.abs()).t()


def _rms(t):
    return float(t.square().mean().sqrt())


def _check(problem, y=None):
    want, mag = _exact(problem)
    terms = problem[0].shape[1] + 32
    err = terms * STEP * mag
    got = (pkg().int4_linear(*problem) if y is None else y).double()
    bad = ~((got - want).abs() <= HALF * (want.abs() + err) + err)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4], got[bad][:4], want[bad][:4], err[bad][:4])
    assert _rms(got - want) <= HALF * _rms(want) + terms**0.5 * STEP * _rms(mag)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("f32", [False, True])
def test_offsets_far_above_the_scales(dev, rows, group, f32):
    _check(_problem(rows, 200, 1024, group, 1.0, f32, seed=rows))


@pytest.mark.parametrize("offset", [None, 0.0, -0.01, -1.0, 30.0])
@pytest.mark.parametrize("rows", [33, 128, 129, 600])
@pytest.mark.parametrize("k, group", [(1056, 32), (640, 128), (4096, 64)])
def test_offsets_and_tables(dev, offset, rows, k, group):
    _check(_problem(rows, 264, k, group, offset, seed=k))


@pytest.mark.parametrize("k", [32, 64, 96, 160, 224])
@pytest.mark.parametrize("rows", [33, 128, 129, 300])
@pytest.mark.parametrize("n", [3, 130])
def test_short_contractions(dev, k, rows, n):
    """Less than a step of columns, and steps that end in a group of 32."""
    _check(_problem(rows, n, k, 32, 1.0, seed=k))


@pytest.mark.parametrize("n", [100, 1000, 8200])
def test_a_row_among_any_number_of_rows(dev, n):
    """A row's results with 1, 17, 33 and 129 rows differ by the rounding of
    FP32 sums and of the results, not of weights: decode continues prefill."""
    import torch

    p = _problem(300, n, 2048, 64, 1.0, seed=n)
    want, mag = _exact((p[0][:1].contiguous(), *p[1:]))
    most = HALF * _rms(want) + (2048 + 32) ** 0.5 * STEP * _rms(mag)
    results = [pkg().int4_linear(p[0][:rows].contiguous(), *p[1:])[:1].double() for rows in (1, 16, 17, 32, 33, 128, 129, 300)]
    for y in results[1:]:
        assert _rms(y - results[0]) <= 2 * most


@pytest.mark.parametrize("rows", [1, 17, 40, 128, 200, 600])
@pytest.mark.parametrize("group", [32, 128])
def test_infinities_and_overflowing_sums(dev, rows, group):
    """Values that the sums of x times codes cannot tell from infinity: the
    formula's own result where it is finite, and its infinity or NaN where it
    is not; rows beside them are left alone."""
    import torch

    p = _problem(rows, 72, 512, group, 0.5, seed=3)
    clean = pkg().int4_linear(*p)
    x = p[0].clone()
    x[0] = 0
    x[0, 9] = float("inf")
    if rows > 3:
        x[1, 5], x[2], x[3] = float("nan"), 0, 0
        x[2, 8], x[3, 500:] = 2.0**127, -(2.0**122)
    y = pkg().int4_linear(x, *p[1:])
    q = torch.stack([p[1] & 15, p[1] >> 4], 2).view(72, 512).double()
    w = q * p[2].double().repeat_interleave(group, 1) + p[3].double().repeat_interleave(group, 1)
    assert torch.equal(y[0].double(), float("inf") * w[:, 9])
    if rows > 3:
        assert y[1].isnan().all()
        for r in (2, 3):
            want = x[r].double() @ w.t()
            assert ((y[r].double() - want).abs() <= 2 * HALF * want.abs()).all()
        assert torch.equal(y[4:], clean[4:])
    scales = p[2].clone()
    scales[7, 0] = float("inf")  # an infinite scale: its output row's own affair
    y = pkg().int4_linear(p[0], p[1], scales, p[3])
    others = [n for n in range(72) if n != 7]
    assert not y[:, 7].isfinite().any() and torch.equal(y[:, others], clean[:, others])


@pytest.mark.parametrize("rows", [17, 129, 400])
def test_quantised_weights_keep_their_codes(dev, rows):
    """quantize_int4 of weights far from zero: the product is that of the
    quantised weights, and as near the weights' own as their codes are."""
    import torch

    M = pkg()
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    w = 1 + 0.01 * torch.randn(136, 512, generator=g, device="cuda")
    x = _problem(rows, 8, 512, 64, 1.0, seed=rows)[0]
    codes, scales, off = M.quantize_int4(w, 64, dtype=torch.float32)
    _check((x, codes, scales, off))
    exact = x.double() @ w.double().t()
    got = M.int4_linear(x, codes, scales, off).double()
    # half a code a weight, and 6 sigma of 15 codes are the group's range
    assert (got - exact).square().mean().sqrt() <= 0.25 * exact.square().mean().sqrt()
