"""GPU tests of the gated MLP against the formulas in 64 bits.

Tolerances: an FP32 sum of K exact products of bf16 values is off by at most
K 2^-24 of the sum of their magnitudes; h, dG and dU are rounded to bf16 once
(half a step, 2^-8 of the value) before they enter a sum, or over at most 16
rows twice, in a high and a low part (2^-16); a result is rounded once more.  sigmoid and exp in FP32 add a few steps of 2^-24, covered by 32.
The magnitudes are summed in 64 bits beside the values.
"""

from __future__ import annotations

import math

import pytest

from conftest import pkg, submodule

pytestmark = pytest.mark.gpu

STEP, HALF = 2.0**-24, 2.0**-8


def _weights(hidden, inter, rows, seed=0, std=0.05, lead=None):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)

    return dict(x=normal(*(lead or (rows,)), hidden), gate=normal(inter, hidden, std=std),
                up=normal(inter, hidden, std=std), down=normal(hidden, inter, std=std),
                dy=normal(*(lead or (rows,)), hidden, std=0.1))


def _formulas(i, limit):
    """{name: (value, error bound before the result's own rounding)}."""
    import torch

    d = {k: v.detach().double() for k, v in i.items()}
    hidden, inter = d["down"].shape
    x, dy = d["x"].reshape(-1, hidden), d["dy"].reshape(-1, hidden)
    rows = x.shape[0]
    op = 2.0**-16 if rows <= 16 else HALF  # rounding of an operand
    limit = math.inf if limit is None else limit
    g, u = x @ d["gate"].t(), x @ d["up"].t()
    eg, eu = (STEP * hidden * (x.abs() @ d[n].abs().t()) for n in ("gate", "up"))
    gc, uc = g.clamp(max=limit), u.clamp(-limit, limit)
    s = torch.sigmoid(gc)
    silu, dsilu = gc * s, s * (1 + gc * (1 - s))
    h = silu * uc
    # |silu'| <= 1.1, |silu''| <= 0.5
    eh = 1.1 * eg * uc.abs() + silu.abs() * eu + 1.1 * eg * eu + 32 * STEP * h.abs()
    rh = op * (h.abs() + eh) + eh  # of h as an operand
    y = h @ d["down"].t()
    ey = rh @ d["down"].abs().t() + STEP * inter * (h.abs() @ d["down"].abs().t())
    dh = dy @ d["down"]
    edh = STEP * hidden * (dy.abs() @ d["down"].abs())
    dg, du = dh * uc * dsilu * (g <= limit), dh * silu * (u.abs() <= limit)
    edg = (edh * (uc.abs() + eu) * (dsilu.abs() + 0.5 * eg) + dh.abs() * (eu * (dsilu.abs() + 0.5 * eg) + uc.abs() * 0.5 * eg)
           + 32 * STEP * (dh * uc).abs())
    edu = edh * (silu.abs() + 1.1 * eg) + dh.abs() * 1.1 * eg + 32 * STEP * du.abs()
    # within the projections' error of the clamp's edge, either side's gradient is right
    if limit < math.inf:
        edg = torch.where((g - limit).abs() <= eg, (dh * uc).abs() * 1.1 + edg, edg)
        edu = torch.where((u.abs() - limit).abs() <= eu, (dh * silu).abs() + edu, edu)
    rg, ru = op * (dg.abs() + edg) + edg, op * (du.abs() + edu) + edu
    dx = dg @ d["gate"] + du @ d["up"]
    edx = rg @ d["gate"].abs() + ru @ d["up"].abs() + STEP * 2 * inter * (
        dg.abs() @ d["gate"].abs() + du.abs() @ d["up"].abs())
    grads = {"x": (dx, edx)}
    for name, (v, e), o in (("gate", (dg, rg), x), ("up", (du, ru), x)):
        grads[name] = (v.t() @ o, e.t() @ o.abs() + STEP * rows * (v.abs().t() @ o.abs()))
    grads["down"] = (dy.t() @ h, dy.abs().t() @ rh + STEP * rows * (dy.abs().t() @ h.abs()))
    return {"y": (y, ey), **grads}


def _near(name, got, want):
    import torch

    value, err = want
    g = got.detach().double().reshape(value.shape)
    bound = HALF * (value.abs() + err) + err + 1e-37
    bad = ~((g - value).abs() <= bound)
    assert not bad.any(), (name, int(bad.sum()), bad.nonzero()[:4], g[bad][:4], value[bad][:4], bound[bad][:4])
    # Those are worst cases of every rounding.  A rounding's error is spread over
    # its half step, rms 2^-8 / sqrt(3) of the value or less, and three of them
    # (operand, operand, result) make 2^-8 of the result's rms; twice that is
    # allowed where there are enough elements for an rms.
    if value.numel() >= 4096:
        assert (g - value).square().mean().sqrt() <= 2 * HALF * value.square().mean().sqrt(), name


def _train(i, limit, fn=None):
    import torch

    leaves = {n: i[n].detach().clone().requires_grad_() for n in ("x", "gate", "up", "down")}
    y = (fn or pkg().gated_mlp)(*leaves.values(), limit)
    return y, dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), i["dy"])))


def _check(i, limit):
    import torch

    want = _formulas(i, limit)
    y, grads = _train(i, limit)
    assert y.shape == i["x"].shape and y.dtype == torch.bfloat16
    _near("y", y, want["y"])
    for name, g in grads.items():
        assert g.shape == i[name].shape and g.dtype == torch.bfloat16
        _near(name, g, want[name])
    with torch.no_grad():
        assert torch.equal(pkg().gated_mlp(i["x"], i["gate"], i["up"], i["down"], limit), y)


@pytest.mark.parametrize("rows", [1, 2, 3, 15, 16, 17, 31, 33, 64, 65, 100, 127, 128, 129, 255, 257, 400, 777])
def test_rows(dev, rows):
    _check(_weights(256, 192, rows, seed=rows), 3.0)


@pytest.mark.parametrize("hidden, inter", [(8, 8), (16, 8), (8, 24), (64, 64), (72, 40), (120, 136), (128, 128), (136, 264),
                                           (256, 8), (8, 512), (520, 1000), (1024, 512), (2048, 1024), (1000, 2056)])
@pytest.mark.parametrize("rows", [1, 50, 300])
def test_widths(dev, hidden, inter, rows):
    _check(_weights(hidden, inter, rows, seed=hidden + inter), None)


@pytest.mark.parametrize("limit", [None, 0.25, 1.0, 10.0])
@pytest.mark.parametrize("rows", [4, 200])
def test_limits(dev, limit, rows):
    _check(_weights(512, 256, rows, std=0.1), limit)


@pytest.mark.parametrize("hidden, inter, rows", [(4096, 1536, 96), (4096, 2048, 1), (1024, 512, 3000), (512, 4096, 1030),
                                                 (4096, 2048, 2050), (7168, 256, 40)])
def test_larger(dev, hidden, inter, rows):
    _check(_weights(hidden, inter, rows, std=0.02), 10.0)


@pytest.mark.parametrize("hidden, inter", [(4096, 2048), (4104, 2048), (4096, 2056), (8, 2048), (4096, 8), (104, 1000)])
@pytest.mark.parametrize("rows", [17, 24, 32])
def test_rows_of_two_mfma_tiles(dev, hidden, inter, rows):
    _check(_weights(hidden, inter, rows, seed=rows, std=0.02), 2.0)


def test_wanted_gradients_alone(dev):
    """Each subset of leaves gets the gradients that all of them get."""
    import itertools

    import torch

    i = _weights(256, 136, 70)
    _, every = _train(i, 2.0)
    for need in itertools.product([False, True], repeat=4):
        if not any(need):
            continue
        leaves = [i[n].detach().clone().requires_grad_(r) for n, r in zip(("x", "gate", "up", "down"), need)]
        y = pkg().gated_mlp(*leaves, 2.0)
        got = torch.autograd.grad(y, [t for t in leaves if t.requires_grad], i["dy"])
        want = [every[n] for n, r in zip(("x", "gate", "up", "down"), need) if r]
        assert all(torch.equal(a, b) for a, b in zip(got, want)), need


# Sizes at which dWd's product, whose sides are the other two's exchanged, is cut into more parts
@pytest.mark.parametrize("rows, hidden, inter", [(3707, 1808, 16), (1436, 16, 1712), (1433, 3976, 32), (900, 64, 4000)])
def test_wanted_gradients_stay_in_their_workspace(dev, monkeypatch, rows, hidden, inter):
    import itertools

    import torch

    i = _weights(hidden, inter, rows)
    native = submodule("_native")
    guards = []

    def workspace(nbytes, device):
        room = torch.full((nbytes + 65536,), 165, dtype=torch.uint8, device=device)
        guards.append(room[nbytes:])
        return room[:nbytes]

    monkeypatch.setattr(native, "workspace", workspace)
    want = _formulas(i, 2.0)
    names = ("x", "gate", "up", "down")
    for need in itertools.product([False, True], repeat=4):
        if not any(need):
            continue
        leaves = [i[n].detach().clone().requires_grad_(r) for n, r in zip(names, need)]
        y = pkg().gated_mlp(*leaves, 2.0)
        got = torch.autograd.grad(y, [t for t in leaves if t.requires_grad], i["dy"])
        for n, g in zip([n for n, r in zip(names, need) if r], got):
            _near(n, g, want[n])
    assert all((g == 165).all() for g in guards)


def test_gradients_against_differences(dev):
    """The slope along a direction in gate, up, down and x against the 64-bit
    formula's difference quotient: what the kernel's gradients are off by is
    their rounding (2 sources of half a step each, as bounds), what the
    quotient is off by its truncation, estimated by halving the step."""
    import torch

    i = _weights(64, 40, 9, seed=5, std=0.2)
    _, grads = _train(i, 4.0)
    want = _formulas(i, 4.0)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    names = ("x", "gate", "up", "down")
    v = {n: torch.randn(i[n].shape, generator=g, device="cuda", dtype=torch.float64) for n in names}

    def quotient(h):
        up = {n: i[n].double() + h * v[n] if n in v else i[n].double() for n in i}
        down = {n: i[n].double() - h * v[n] if n in v else i[n].double() for n in i}
        f = [float((_formulas(j, 4.0)["y"][0] * i["dy"].double()).sum()) for j in (up, down)]
        return (f[0] - f[1]) / (2 * h)

    a, b = quotient(1e-4), quotient(5e-5)
    slope = sum(float((grads[n].double() * v[n]).sum()) for n in names)
    noise = sum(float(((HALF * (want[n][0].abs() + want[n][1]) + want[n][1]) * v[n].abs()).sum()) for n in names)
    assert abs(slope - b) <= noise + 4 * abs(a - b) + 1e-6 * abs(b)


def test_nan_and_infinity_stay_in_their_rows(dev):
    import torch

    i = _weights(256, 128, 40)
    clean = pkg().gated_mlp(i["x"], i["gate"], i["up"], i["down"], 3.0)
    x = i["x"].clone()
    x[7, 3], x[20, 100], x[39, 255] = float("nan"), float("inf"), float("-inf")
    y = pkg().gated_mlp(x, i["gate"], i["up"], i["down"], 3.0)
    assert y[7].isnan().all()
    keep = [r for r in range(40) if r not in (7, 20, 39)]
    assert torch.equal(y[keep], clean[keep])


def test_rows_do_not_depend_on_their_number(dev):
    """Rows behind a batch's last are not touched, and views and strides give
    what copies give."""
    import torch

    M = pkg()
    i = _weights(256, 128, 33)
    flat = torch.empty(33 * 256 + 1, device=dev, dtype=torch.bfloat16)
    flat[1:].view(33, 256).copy_(i["x"])
    stacked = torch.cat([i["gate"], i["up"]])
    want = M.gated_mlp(i["x"], i["gate"], i["up"], i["down"])
    assert torch.equal(M.gated_mlp(flat[1:].view(33, 256), stacked[:128], stacked[128:], i["down"]), want)
    assert torch.equal(M.gated_mlp(i["x"].t().contiguous().t(), i["gate"].t().contiguous().t(), i["up"],
                                   i["down"].t().contiguous().t()), want)
    assert torch.equal(M.gated_mlp(i["x"].view(3, 11, 256), i["gate"], i["up"], i["down"]), want.view(3, 11, 256))


def test_empty(dev):
    import torch

    i = _weights(64, 32, 4)
    x = i["x"][:0].requires_grad_()
    w = [i[n].requires_grad_() for n in ("gate", "up", "down")]
    y = pkg().gated_mlp(x, *w)
    assert y.shape == (0, 64)
    grads = torch.autograd.grad(y, [x, *w], torch.zeros_like(y))
    assert all(g.shape == t.shape and (g == 0).all() for g, t in zip(grads, [x, *w]))


def test_runs_repeat(dev):
    import torch

    for shape in ((256, 136, 900), (512, 256, 20)):
        i = _weights(*shape)
        y, grads = _train(i, 2.0)
        for _ in range(3):
            y2, again = _train(i, 2.0)
            assert torch.equal(y, y2) and all(torch.equal(grads[n], again[n]) for n in grads)


@pytest.mark.parametrize("rows", [1, 70, 300])
def test_other_stream_and_captured_graph(dev, rows):
    import torch

    gated = submodule("gated")
    i = _weights(256, 128, rows)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())

    def both():
        args = (i["x"], i["gate"], i["up"], i["down"])
        y, *kept = gated.native_gated_mlp(*args, 2.0, True)
        z = gated.native_gated_mlp(*args, 2.0, False)[0]
        return [y, z] + gated.native_gated_mlp_backward(*args, *kept, i["dy"], 2.0, [True] * 4)

    with torch.cuda.stream(s):
        both()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = both()
    torch.cuda.current_stream().wait_stream(s)
    for k in range(3):
        fresh = _weights(256, 128, rows, seed=30 + k)
        for n in fresh:
            i[n].copy_(fresh[n])
        graph.replay()
        torch.cuda.synchronize()
        want = both()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_traced_call_equals_eager(dev):
    import torch

    i = _weights(128, 64, 20)
    y, grads = _train(i, 2.0)
    M = pkg()
    compiled = torch.compile(lambda *a: M.gated_mlp(*a), backend="aot_eager", fullgraph=True)
    cy, cgrads = _train(i, 2.0, fn=compiled)
    assert torch.equal(y, cy) and all(torch.equal(grads[n], cgrads[n]) for n in grads)


def test_module_trains(dev):
    """GatedMLP's parameters get gated_mlp's gradients."""
    import torch

    M = pkg()
    m = M.GatedMLP(128, 64, limit=3.0, device=dev)
    x = torch.randn(5, 7, 128, device=dev).to(torch.bfloat16)
    dy = torch.randn(5, 7, 128, device=dev).to(torch.bfloat16)
    m(x).backward(dy)
    leaves = [p.detach().clone().requires_grad_() for p in (m.gate_proj.weight, m.up_proj.weight, m.down_proj.weight)]
    want = torch.autograd.grad(M.gated_mlp(x, *leaves, 3.0), leaves, dy)
    for p, w in zip((m.gate_proj.weight, m.up_proj.weight, m.down_proj.weight), want):
        assert torch.equal(p.grad, w)


def test_refusals(dev):
    import torch

    M = pkg()
    i = _weights(64, 32, 4)
    x, g, u, d = i["x"], i["gate"], i["up"], i["down"]
    bad = [
        lambda: M.gated_mlp(x.float(), g, u, d), lambda: M.gated_mlp(x, g.half(), u, d), lambda: M.gated_mlp(x, g, u[:16], d),
        lambda: M.gated_mlp(x, g, u, d.t()), lambda: M.gated_mlp(x[:, :32], g, u, d), lambda: M.gated_mlp(x, g, u, d, 0.0),
        lambda: M.gated_mlp(x, g, u, d, -1.0), lambda: M.gated_mlp(x, g, u, d, float("nan")),
        lambda: M.gated_mlp(x[:, :60], g[:, :60], u[:, :60], d[:60]), lambda: M.gated_mlp(x, g[:28], u[:28], d[:, :28]),
        lambda: M.gated_mlp(x, g[:0], u[:0], d[:, :0]), lambda: M.gated_mlp(x, g.cpu(), u, d),
        lambda: M.gated_mlp(x, g[0], u[0], d[0]),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {k} was not refused")


def test_offsets_past_32_bits(dev):
    """G, U and h of more than 2^32 bytes, and the widest operand the kernels
    address from one tile: the last rows are those of a call of their own."""
    import torch

    M = pkg()
    rows, hidden, inter, tail = 270_000, 64, 8192, 40
    i = _weights(hidden, inter, tail, std=0.05)
    x = torch.randn(tail, hidden, device=dev).to(torch.bfloat16).repeat(rows // tail, 1)
    x[-tail:] = i["x"]
    dy = torch.zeros(rows, hidden, device=dev, dtype=torch.bfloat16)
    dy[-tail:] = i["dy"]
    leaves = [x.requires_grad_(), *(i[n].clone().requires_grad_() for n in ("gate", "up", "down"))]
    y = M.gated_mlp(*leaves, 4.0)
    grads = torch.autograd.grad(y, leaves, dy)
    want = _formulas(i, 4.0)
    _near("y", y[-tail:], want["y"])
    _near("x", grads[0][-tail:], want["x"])
    assert (grads[0][:-tail] == 0).all()
    # rows without a gradient add zeros: the sums are the last rows', in other parts
    for n, g in zip(("gate", "up", "down"), grads[1:]):
        _near(n, g, want[n])
    wide = 1 << 17
    j = _weights(wide, 8, 300, std=0.003)
    y = M.gated_mlp(j["x"], j["gate"], j["up"], j["down"])
    _near("y", y, _formulas(j, None)["y"])


def test_no_second_derivative_is_claimed(dev):
    import torch

    i = _weights(64, 32, 4)
    x = i["x"].requires_grad_()
    g, = torch.autograd.grad(pkg().gated_mlp(x, i["gate"], i["up"], i["down"]).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_two_streams_at_once(dev):
    """Calls that overlap on two streams have their own workspaces."""
    import torch

    M = pkg()
    problems = [_weights(512, 256, rows, seed=rows) for rows in (90, 700)]
    want = [_train(i, 2.0) for i in problems]
    streams = [torch.cuda.Stream() for _ in problems]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, i in zip(streams, problems):
            with torch.cuda.stream(s):
                got.append(_train(i, 2.0))
    torch.cuda.synchronize()
    for k, (y, grads) in enumerate(got):
        wy, wg = want[k % 2]
        assert torch.equal(y, wy) and all(torch.equal(grads[n], wg[n]) for n in wg), k
