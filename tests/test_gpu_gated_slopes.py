"""GPU tests of each of the gated MLP's gradients against difference quotients,
one input at a time.

The input moves along the formula's own normalised gradient, so the slope is
that gradient's length.  What the kernel's gradient may be off by: its
elements' error bounds are those of the gated MLP's other tests (half a step of
bf16 for the result, and the errors of its operands and sums); errors of either
sign add up to a few roots of the summed squares, of which 4 are allowed.  A
gradient without a part of its terms, halved or zero is far outside: the test
asks that the allowance is below a fiftieth of the slope."""

from __future__ import annotations

import pytest

from test_gpu_gated import HALF, _formulas, _train, _weights

NAMES = ("x", "gate", "up", "down")


def _slope(i, limit, name):
    """(direction, slope by the formula, its difference quotient in 64 bits and
    that quotient's own error, allowance for a kernel's gradient)."""
    value, err = _formulas(i, limit)[name]
    length = float(value.norm())
    v = value / length

    def loss(h):
        moved = {n: t.double() for n, t in i.items()}
        moved[name] = moved[name] + h * v.view(moved[name].shape)
        dy = i["dy"].double().reshape(-1, i["dy"].shape[-1])
        return float((_formulas(moved, limit)["y"][0] * dy).sum())

    a, b = ((loss(h) - loss(-h)) / (2 * h) for h in (1e-4, 5e-5))
    noise = 4 * float((((HALF * (value.abs() + err) + err) * v) ** 2).sum().sqrt())
    return v, length, b, 4 * abs(a - b) + 1e-7 * abs(b), noise


# (a clamp's edge is a kink: with one, the quotient may differ on either side of it)
@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 9, 16, 17, 70])
@pytest.mark.parametrize("limit", [None, 4.0])
@pytest.mark.parametrize("name", NAMES)
def test_gradient_along_itself(dev, rows, limit, name):
    i = _weights(64, 40, rows, seed=rows, std=0.2)
    v, length, quotient, truncation, noise = _slope(i, limit, name)
    assert abs(length - quotient) <= truncation
    assert noise <= length / 50
    got = _train(i, limit)[1][name].double().reshape(v.shape)
    assert abs(float((got * v).sum()) - quotient) <= noise + truncation


def _rounded_where_said(i, limit):
    """The formulas in 64 bits with the roundings that the operator names and no
    others: dG, dU and the gradients' h to bf16 as operands above 16 rows, the
    output's h above 32 (over at most 4,096 hidden and 2,048 intermediate columns)."""
    import math

    import torch

    d = {n: t.double() for n, t in i.items()}
    limit = math.inf if limit is None else limit

    def operand(t, exact_rows=16):
        return t if i["x"].shape[0] <= exact_rows else t.to(torch.bfloat16).double()

    g, u = d["x"] @ d["gate"].t(), d["x"] @ d["up"].t()
    gc, uc = g.clamp(max=limit), u.clamp(-limit, limit)
    s = torch.sigmoid(gc)
    h = gc * s * uc
    dh = d["dy"] @ d["down"]
    dg = operand(dh * uc * s * (1 + gc * (1 - s)) * (g <= limit))
    du = operand(dh * gc * s * (u.abs() <= limit))
    return {"y": operand(h, 32) @ d["down"].t(), "x": dg @ d["gate"] + du @ d["up"], "gate": dg.t() @ d["x"], "up": du.t() @ d["x"],
            "down": d["dy"].t() @ operand(h)}


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [16, 17, 32, 33, 70, 300])
def test_no_rounding_but_those_named(dev, rows):
    """Beside those roundings a result has one of its own, of at most half a
    step 2^-8 of its value and spread over it: an rms of 2^-8 / sqrt(3) of the
    result's at most (FP32 sums add less than a hundredth of that).  One rounding
    more would have an rms of sqrt(2) times what one has in fact, three
    quarters of that bound."""
    import torch

    i = _weights(512, 256, rows, seed=rows)
    want = _rounded_where_said(i, 3.0)
    y, grads = _train(i, 3.0)
    for name, got in {"y": y, **grads}.items():
        far = (got.double() - want[name]).square().mean().sqrt() / want[name].square().mean().sqrt()
        assert far <= 1.01 * HALF / 3**0.5, (name, float(far))
        if rows > 16:  # the bound sees a rounding more: of the results, once to a neighbour's precision
            twice = (want[name] * (1 + HALF * (torch.rand_like(want[name]) * 2 - 1))).to(torch.bfloat16).double()
            more = (twice - want[name]).square().mean().sqrt() / want[name].square().mean().sqrt()
            assert more > 1.01 * HALF / 3**0.5
