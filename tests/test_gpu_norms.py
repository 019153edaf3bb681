"""GPU tests of rms_norm and residual_norm against the formulas in 64 bits.

Tolerances: a result is off by its own rounding, half a step of its type
relative to the value, and by FP32 arithmetic, 2^-24 a step relative to the
magnitudes that were added.  A row's sum is a chain of at most 16 + 6 + 16
additions and enters a value through a square root, so 64 steps of the summed
magnitudes cover each elementwise result; a column sum adds `rows` terms.
"""

from __future__ import annotations

import math

import pytest

from conftest import pkg, submodule

pytestmark = pytest.mark.gpu

STEP = 2.0**-24


def _half(dtype):
    import torch

    return torch.finfo(dtype).eps / 2


def _near(got, want, mag, steps=64):
    import torch

    assert got.shape == want.shape
    g = got.detach().double()
    bound = _half(got.dtype) * (want.abs() + STEP * steps * mag) + STEP * steps * mag
    bad = ~((g - want).abs() <= bound)
    bad &= ~(torch.isnan(g) & torch.isnan(want)) & ~((g == want))
    assert not bad.any(), (int(bad.sum()), (g - want).abs()[bad][:4], bound[bad][:4], bad.nonzero()[:4])


def _types(name):
    import torch

    return {"b": torch.bfloat16, "f": torch.float32}[name]


def _inputs(rows, width, types, gate, seed=0, lead=None):
    """residual, out, post, gate, next, d_new, d_y on the device."""
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0, t="f"):
        return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(_types(t))

    lead = lead or (rows,)
    shape = (*lead, width)
    gates = {"none": None, "channel": (width,), "token": (*lead, 1), "full": shape, "one": (1,), "scalar": (),
             "sequence": (lead[0], *([1] * (len(lead) - 1)), width), "sequence one": (lead[0],) + (1,) * len(lead),
             "inner": (1,) * (len(lead) - 1) + (lead[-1], width)}[gate]
    return dict(
        residual=normal(*shape, std=2.0, t=types[0]), out=normal(*shape, std=0.5, mean=0.1, t=types[1]),
        post=normal(width, std=0.2, mean=1.0, t=types[2]),
        gate=None if gates is None else normal(*gates, std=0.5, mean=0.5, t=types[2]),
        next=normal(width, std=0.2, mean=1.0, t=types[2]),
        d_new=normal(*shape, std=0.3, t=types[0]), d_y=normal(*shape, std=0.3, t=types[1]))


def _formulas(i, scale, eps, post_norm=True):
    """Outputs, gradients, and the magnitudes that each adds, in 64 bits."""
    import torch

    width = i["residual"].shape[-1]
    d = {k: None if v is None else v.detach().double() for k, v in i.items()}
    x, o = d["residual"], d["out"]
    gate = d["gate"] if d["gate"] is not None else torch.ones((), dtype=torch.float64, device=x.device)
    p = d["post"] if post_norm else torch.ones((), dtype=torch.float64, device=x.device)
    ro = 1 / (o.square().mean(-1, keepdim=True) + eps).sqrt() if post_norm else torch.ones_like(o[..., :1])
    oh = o * ro
    s = oh * p
    new = x + scale * gate * s
    new_mag = x.abs() + (scale * gate * s).abs()
    r = 1 / (new.square().mean(-1, keepdim=True) + eps).sqrt()
    xh = new * r
    xh_mag = new_mag * r + xh.abs()  # r is as exact as the values it is made of
    y = xh * d["next"]
    t = d["d_y"] * d["next"]
    dot = (t * xh).mean(-1, keepdim=True)
    dot_mag = (t.abs() * xh_mag).mean(-1, keepdim=True)
    dx = d["d_new"] + r * (t - xh * dot)
    dx_mag = d["d_new"].abs() + r * (t.abs() + xh_mag * dot_mag)
    ds, ds_mag = scale * gate * dx, (scale * gate).abs() * dx_mag
    dg, dg_mag = scale * s * dx, (scale * s).abs() * dx_mag
    if post_norm:
        q, q_mag = p * ds, p.abs() * ds_mag
        do = ro * (q - oh * (q * oh).mean(-1, keepdim=True))
        do_mag = ro * (q_mag + oh.abs() * (q_mag * oh.abs()).mean(-1, keepdim=True))
    else:
        do, do_mag = ds, ds_mag
    rows = range(x.dim() - 1)
    got = dict(new=(new, new_mag), y=(y, xh_mag * d["next"].abs()), residual=(dx, dx_mag), out=(do, do_mag),
               next=((d["d_y"] * xh).sum(tuple(rows)), (d["d_y"].abs() * xh_mag).sum(tuple(rows))),
               post=((ds * oh).sum(tuple(rows)), (ds_mag * oh.abs()).sum(tuple(rows))))
    if d["gate"] is not None:
        got["gate"] = tuple(v.sum_to_size(d["gate"].shape) for v in (dg, dg_mag))
    return got


def _train(i, scale, eps, post_norm=True, fn=None):
    import torch

    leaves = {k: v.detach().clone().requires_grad_() for k, v in i.items() if v is not None and not k.startswith("d_")}
    if not post_norm:
        leaves.pop("post")
    fn = fn or pkg().residual_norm
    x, y = fn(leaves["residual"], leaves["out"], post_weight=leaves.get("post"), gate=leaves.get("gate"), scale=scale,
              next_weight=leaves["next"], eps=eps)
    grads = torch.autograd.grad([x, y], list(leaves.values()), [i["d_new"], i["d_y"]])
    return x, y, dict(zip(leaves, grads))


def _check(i, scale, eps, post_norm=True, rows=None):
    import torch

    want = _formulas(i, scale, eps, post_norm)
    x, y, grads = _train(i, scale, eps, post_norm)
    assert x.dtype == i["residual"].dtype and y.dtype == i["out"].dtype
    _near(x, *want["new"])
    _near(y, *want["y"])
    rows = i["residual"].numel() // i["residual"].shape[-1]
    for name, g in grads.items():
        assert g.dtype == i[name].dtype
        summed = name in ("next", "post") or (name == "gate" and i["gate"].numel() < i["residual"].numel())
        terms = rows + i["residual"].shape[-1] if summed else 0
        _near(g, *want[name], steps=64 + terms)
    with torch.no_grad():  # the forward alone gives the same values
        x0, y0 = pkg().residual_norm(i["residual"], i["out"], post_weight=i["post"] if post_norm else None,
                                     gate=i["gate"], scale=scale, next_weight=i["next"], eps=eps)
    assert torch.equal(x0, x) and torch.equal(y0, y)


@pytest.mark.parametrize("width", [1, 7, 64, 511, 512, 520, 1001, 2048, 2049, 4096, 5000, 8191, 8192, 9001, 12288, 16383, 16384])
def test_widths(dev, width):
    _check(_inputs(5, width, "bbb", "channel"), 0.5, 1e-6)


@pytest.mark.parametrize("types", ["bbb", "bbf", "fbb", "fbf", "ffb", "fff", "bff"])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full", "one", "scalar"])
def test_types_and_gates(dev, types, gate):
    _check(_inputs(37, 264, types, gate), 0.25, 1e-5)


@pytest.mark.parametrize("gate", ["sequence", "sequence one", "inner", "token", "channel"])
@pytest.mark.parametrize("lead", [(3, 11), (1, 5), (600, 2), (2, 3, 4)])
def test_gates_over_sequences(dev, gate, lead):
    _check(_inputs(math.prod(lead), 40, "bbb", gate, lead=lead), 1.0, 1e-6)


@pytest.mark.parametrize("rows", [1, 2, 511, 512, 513, 1025, 3001])
def test_rows(dev, rows):
    _check(_inputs(rows, 72, "fbf", "channel"), 1.0, 1e-6)


def test_without_post_norm(dev):
    for gate in ("none", "channel", "token", "full"):
        _check(_inputs(19, 136, "bbb", gate), -0.5, 1e-6, post_norm=False)


def test_without_next_norm(dev):
    import torch

    i = _inputs(9, 96, "fbb", "channel")
    leaves = [i[n].clone().requires_grad_() for n in ("residual", "out", "post", "gate")]
    x, y = pkg().residual_norm(leaves[0], leaves[1], post_weight=leaves[2], gate=leaves[3], scale=0.5)
    assert y is None
    grads = torch.autograd.grad(x, leaves, i["d_new"])
    j = dict(i, d_y=torch.zeros_like(i["d_y"]))
    want = _formulas(j, 0.5, 1e-6)
    _near(x, *want["new"])
    for g, name in zip(grads, ("residual", "out", "post", "gate")):
        _near(g, *want[name], steps=200)


@pytest.mark.parametrize("types", ["bb", "fb", "bf", "ff"])
@pytest.mark.parametrize("width", [5, 512, 4096])
def test_rms_norm(dev, types, width):
    import torch

    i = _inputs(33, width, types + "b", "none")
    x, w = i["residual"].clone().requires_grad_(), i["next"].clone().requires_grad_()
    y = pkg().rms_norm(x, w, 1e-5, dtype=_types(types[1]))
    gx, gw = torch.autograd.grad(y, [x, w], i["d_y"])
    j = dict(i, out=torch.zeros_like(i["out"]), d_new=torch.zeros_like(i["d_new"]))
    want = _formulas(j, 0.0, 1e-5)
    _near(y, *want["y"])
    _near(gx, *want["residual"])
    _near(gw, *want["next"], steps=128)
    assert torch.equal(pkg().rms_norm(i["residual"], None, dtype=torch.float32),
                       pkg().rms_norm(i["residual"], torch.ones_like(w), dtype=torch.float32))


def test_gradients_against_differences(dev):
    """<gradient, v> against (L(+h) - L(-h)) / 2h for every input at once.  The
    quotient's truncation is the same quotient's in 64 bits; its noise is the
    FP32 error of the outputs over h."""
    import torch

    i = _inputs(6, 48, "fff", "token", seed=3)
    names = ("residual", "out", "post", "gate", "next")
    g = torch.Generator(device="cuda")
    g.manual_seed(11)
    v = {n: torch.randn(i[n].shape, generator=g, device="cuda") for n in names}
    h = 2.0**-7

    def loss(j, kernel):
        if kernel:
            x, y = pkg().residual_norm(j["residual"], j["out"], post_weight=j["post"], gate=j["gate"], scale=0.5,
                                       next_weight=j["next"], eps=1e-3)
        else:
            f = _formulas(j, 0.5, 1e-3)
            x, y = f["new"][0], f["y"][0]
        return float((x.double() * i["d_new"].double()).sum() + (y.double() * i["d_y"].double()).sum())

    # moved inputs that are exact in FP32 for both sides
    up = dict(i, **{n: i[n] + h * v[n] for n in names})
    down = dict(i, **{n: i[n] - h * v[n] for n in names})
    moved = {n: (up[n].double() - down[n].double()) / (2 * h) for n in names}
    _, _, grads = _train(i, 0.5, 1e-3)
    slope = sum(float((grads[n].double() * moved[n]).sum()) for n in names)
    want = _formulas(i, 0.5, 1e-3)
    exact = sum(float((want[n][0] * moved[n]).sum()) for n in names)
    quotient, quotient64 = ((loss(up, k) - loss(down, k)) / (2 * h) for k in (True, False))
    mags = sum(float((want[a][1] * i[b].double().abs()).sum()) for a, b in (("new", "d_new"), ("y", "d_y")))
    assert abs(quotient - quotient64) <= 2 * 64 * STEP * mags / h
    grad_mag = sum(float((want[n][1] * moved[n].abs()).sum()) for n in names)
    assert abs(slope - exact) <= 256 * STEP * grad_mag
    assert abs(slope - quotient) <= abs(exact - quotient64) + 2 * 64 * STEP * mags / h + 256 * STEP * grad_mag


def test_large_and_special_values(dev):
    """Rows of zeros, of one infinity, of NaN, and of the type's largest
    values, beside an ordinary row that they must leave alone."""
    import torch

    M = pkg()
    w = torch.ones(64, device=dev, dtype=torch.bfloat16)
    x = torch.randn(6, 64, device=dev).to(torch.bfloat16)
    x[0] = 0
    x[1, 3] = float("inf")
    x[2, 5] = float("nan")
    x[3] = 2.0**63  # squares sum to infinity in FP32, as in the formula in 32 bits
    y = M.rms_norm(x, w, 1e-6).float()
    assert (y[0] == 0).all()
    assert y[1, 3].isnan() and (y[1, :3] == 0).all() and (y[1, 4:] == 0).all()
    assert y[2].isnan().all()
    want = x[4:].double() / (x[4:].double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
    _near(y[4:].to(torch.bfloat16), want, want.abs())
    assert M.rms_norm(torch.zeros(2, 64, device=dev), None, 0.0).isnan().all()


def test_empty(dev):
    import torch

    M = pkg()
    x = torch.zeros(0, 3, 16, device=dev, dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(16, device=dev, requires_grad=True)
    g = torch.ones(16, device=dev, requires_grad=True)
    a, b = M.residual_norm(x, x.detach(), post_weight=w, gate=g, next_weight=w)
    assert a.shape == b.shape == x.shape
    (a.sum() + b.float().sum()).backward()
    assert x.grad.shape == x.shape and (w.grad == 0).all() and (g.grad == 0).all()


def test_strides_views_and_offsets(dev):
    """Transposed, sliced and 2-byte aligned tensors give what their copies give."""
    import torch

    M = pkg()
    base = torch.randn(24, 18, device=dev).to(torch.bfloat16)
    flat = torch.randn(24 * 16 + 1, device=dev).to(torch.bfloat16)
    views = [base.t()[:, :16], base[:, 1:17], flat[1:].view(24, 16), base[::2, :16]]
    for v in views:
        o = torch.randn(v.shape, device=dev).to(torch.bfloat16).t().contiguous().t()
        assert not (v.is_contiguous() and o.is_contiguous())
        w = flat[3:3 + v.shape[-1]]
        a, b = M.residual_norm(v, o, post_weight=w, next_weight=w)
        c, d = M.residual_norm(v.clone(memory_format=torch.contiguous_format),
                               o.clone(memory_format=torch.contiguous_format), post_weight=w.clone(),
                               next_weight=w.clone())
        assert torch.equal(a, c) and torch.equal(b, d)


def test_runs_and_orders_repeat(dev):
    """The same bits on every run: no sum depends on what ran first."""
    import torch

    i = _inputs(2049, 520, "bbb", "channel")
    first = _train(i, 0.5, 1e-6)
    for _ in range(3):
        again = _train(i, 0.5, 1e-6)
        assert torch.equal(first[0], again[0]) and all(torch.equal(first[2][n], again[2][n]) for n in first[2])


def test_other_stream_and_captured_graph(dev):
    """On a stream of its own, and captured forward and backward (native calls)
    replayed with new values between eager work."""
    import torch

    M, norms = pkg(), submodule("norms")
    N = submodule("_native")
    i = _inputs(65, 520, "bbb", "channel")
    args = (i["residual"], i["out"], i["post"], i["gate"], i["next"])
    form = (N.GATE_COLUMNS, 65, 0.5, 1e-6)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())

    def both():
        x, y, stats = norms.native_residual_norm(*args, *form, True, False)
        return [x, y] + norms.native_residual_norm_backward(*args, stats, i["d_new"], i["d_y"], *form, False, [True] * 5)

    with torch.cuda.stream(s):
        both()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = both()
    torch.cuda.current_stream().wait_stream(s)
    for k in range(3):
        fresh = _inputs(65, 520, "bbb", "channel", seed=20 + k)
        for n in fresh:
            i[n].copy_(fresh[n])
        graph.replay()
        torch.cuda.synchronize()
        want = both()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


def test_traced_call_equals_eager(dev):
    """torch.compile traces the calls as ops, with their gradients."""
    import torch

    i = _inputs(12, 64, "fbb", "token")
    x, y, grads = _train(i, 0.5, 1e-6)
    M = pkg()

    def fn(residual, out, **kw):
        return M.residual_norm(residual, out, **kw)

    compiled = torch.compile(fn, backend="aot_eager", fullgraph=True)
    cx, cy, cgrads = _train(i, 0.5, 1e-6, fn=compiled)
    assert torch.equal(x, cx) and torch.equal(y, cy) and all(torch.equal(grads[n], cgrads[n]) for n in grads)


def test_refusals(dev):
    import torch

    M = pkg()
    x = torch.zeros(4, 16, device=dev, dtype=torch.bfloat16)
    w = torch.ones(16, device=dev)
    bad = [
        lambda: M.rms_norm(x.half(), w), lambda: M.rms_norm(x, w.half()), lambda: M.rms_norm(x, w[:8]),
        lambda: M.rms_norm(x, w.view(1, 16)), lambda: M.rms_norm(x, w, dtype=torch.float16),
        lambda: M.rms_norm(x[:, :0], None), lambda: M.rms_norm(x, w.cpu()), lambda: M.rms_norm(x, w, -1.0),
        lambda: M.rms_norm(torch.zeros(2, 16385, device=dev)),
        lambda: M.residual_norm(x, x[:2]), lambda: M.residual_norm(x, x.half()),
        lambda: M.residual_norm(x, x, gate=w[:8]), lambda: M.residual_norm(x, x, gate=torch.ones(3, 1, device=dev)),
        lambda: M.residual_norm(x, x, gate=torch.ones(1, 4, 16, device=dev)),
        lambda: M.residual_norm(x, x, gate=w.half()), lambda: M.residual_norm(x, x, post_weight=w[:4]),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {k} was not refused")


@pytest.mark.parametrize("width", [5, 64, 100, 1001, 2050, 5003, 9001])
@pytest.mark.parametrize("post_norm", [True, False])
def test_in_place(dev, width, post_norm):
    """The C entry points where an output is an input's own memory: the new
    residual over residual or out, y over out or residual, d_residual over
    d_new_residual; each gives the bits of separate memory."""
    import ctypes

    import torch

    N, norms = submodule("_native"), submodule("norms")
    i = _inputs(7, width, "bbb", "none", seed=width)
    post = i["post"] if post_norm else None
    form = (N.GATE_NONE, 1, 0.5, 1e-6)
    x, y, stats = norms.native_residual_norm(i["residual"], i["out"], post, None, i["next"], *form, True, False)
    alone = norms.native_residual_norm(i["residual"], None, None, None, i["next"], N.GATE_NONE, 1, 1.0, 1e-6, True, False)[1]

    def call(residual, out, new, normed):
        n = N.Norm(rows=7, width=width, rows_per_gate=1, residual=residual.data_ptr(), next_weight=i["next"].data_ptr(),
                   out=None if out is None else out.data_ptr(), new_residual=None if new is None else new.data_ptr(),
                   post_weight=None if post is None or out is None else post.data_ptr(), y=normed.data_ptr(),
                   post_norm=int(post is not None and out is not None), scale=0.5, eps=1e-6)
        N.run(residual.get_device(), N.lib().glm53_residual_norm, ctypes.byref(n))

    for new_at, y_at in (("residual", "out"), ("out", "fresh"), ("residual", "fresh"), ("fresh", "out")):
        t = dict(residual=i["residual"].clone(), out=i["out"].clone(), fresh=torch.empty_like(i["out"]))
        call(t["residual"], t["out"], t[new_at], t[y_at])
        assert torch.equal(t[new_at], x) and torch.equal(t[y_at], y), (new_at, y_at)
    t = i["residual"].clone()
    call(t, None, None, t)
    assert torch.equal(t, alone)

    for d_y in (i["d_y"], None):
        want = norms.native_residual_norm_backward(i["residual"], i["out"], post, None, i["next"], stats, i["d_new"], d_y,
                                                   *form, False, [True, True, False, False, False])
        d = i["d_new"].clone()
        d_out = torch.empty_like(i["out"])
        ws = torch.empty(N.lib().glm53_residual_norm_workspace_bytes(7, width, 1), dtype=torch.uint8, device=dev)
        n = N.Norm(rows=7, width=width, rows_per_gate=1, residual=i["residual"].data_ptr(), out=i["out"].data_ptr(),
                   post_weight=None if post is None else post.data_ptr(), next_weight=i["next"].data_ptr(),
                   stats=stats.data_ptr(), d_new_residual=d.data_ptr(), d_y=None if d_y is None else d_y.data_ptr(),
                   d_residual=d.data_ptr(), d_out=d_out.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(),
                   post_norm=int(post is not None), scale=0.5, eps=1e-6)
        N.run(d.get_device(), N.lib().glm53_residual_norm_backward, ctypes.byref(n))
        assert torch.equal(d, want[0]) and torch.equal(d_out, want[1])


def test_offsets_past_32_bits(dev):
    """Tensors of more than 2^31 elements: the last rows are those of a call of
    their own, forward and backward."""
    import torch

    M = pkg()
    rows, width, tail = 140_000, 16384, 3
    assert rows * width > 2**31
    i = _inputs(tail, width, "bbb", "channel", seed=2)
    big = {n: torch.zeros(rows, width, device=dev, dtype=torch.bfloat16) for n in ("residual", "out", "d_new", "d_y")}
    for n in big:
        big[n][-tail:] = i[n]
    big["out"][:-tail, 0] = 1  # rows that are not all zero
    big["residual"].requires_grad_()
    big["out"].requires_grad_()
    w = {n: i[n].clone().requires_grad_() for n in ("post", "gate", "next")}
    x, y = M.residual_norm(big["residual"], big["out"], post_weight=w["post"], gate=w["gate"], scale=0.5,
                           next_weight=w["next"])
    grads = torch.autograd.grad([x, y], [big["residual"], big["out"], *w.values()], [big["d_new"], big["d_y"]])
    want = _formulas(i, 0.5, 1e-6)
    _near(x[-tail:], *want["new"])
    _near(y[-tail:], *want["y"])
    _near(grads[0][-tail:], *want["residual"])
    _near(grads[1][-tail:], *want["out"])
    for n, g in zip(("post", "gate", "next"), grads[2:]):
        _near(g, *want[n], steps=200)


def test_more_rows_than_one_grid(dev):
    """2^26 rows of 64 threads are the 2^32 that a grid may not have."""
    import torch

    M = pkg()
    rows, width = 2**26 + 1025, 8
    x = torch.randn(rows // 64 + 1, width, device=dev).to(torch.bfloat16).repeat(64, 1)[:rows]
    period = x[:rows // 64 + 1]
    got = M.rms_norm(x)
    want = M.rms_norm(period)
    d = period.double()
    value = d / (d.square().mean(1, keepdim=True) + 1e-6).sqrt()
    _near(want, value, value.abs(), steps=width + 8)
    for first in range(0, rows, len(period)):
        part = got[first:first + len(period)]
        assert torch.equal(part, want[:len(part)]), first


def test_no_second_derivative_is_claimed(dev):
    import torch

    x = torch.randn(3, 16, device=dev, requires_grad=True)
    g, = torch.autograd.grad(pkg().rms_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_one_gradient_given_or_wanted(dev):
    """Only the new residual's, or only y's gradient comes; each subset of
    leaves gets what all of them get."""
    import itertools

    import torch

    M = pkg()
    i = _inputs(21, 72, "fbf", "token", seed=4)
    names = ("residual", "out", "post", "gate", "next")

    def run(need, given):
        t = [i[n].detach().clone().requires_grad_(r) for n, r in zip(names, need)]
        x, y = M.residual_norm(t[0], t[1], post_weight=t[2], gate=t[3], scale=0.5, next_weight=t[4])
        pairs = [p for p, g in zip(((x, i["d_new"]), (y, i["d_y"])), given) if g]
        wanted = [v for v in t if v.requires_grad]
        got = torch.autograd.grad([p[0] for p in pairs], wanted, [p[1] for p in pairs], allow_unused=True)
        return dict(zip([n for n, r in zip(names, need) if r], got))

    for given in ((True, True), (True, False), (False, True)):
        j = dict(i)
        for n, g in zip(("d_new", "d_y"), given):
            if not g:
                j[n] = torch.zeros_like(i[n])
        want = _formulas(j, 0.5, 1e-6)
        every = run([True] * 5, given)
        for n, g in every.items():
            if g is None:
                assert n == "next" and not given[1]
            else:
                _near(g, *want[n], steps=200)
        for need in itertools.product([False, True], repeat=5):
            if any(need) and not (need == (False,) * 4 + (True,) and not given[1]):
                got = run(need, given)
                assert all((g is None and every[n] is None) or torch.equal(g, every[n]) for n, g in got.items()), need
