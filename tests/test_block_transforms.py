"""What forward mode and torch.func get from the dense block's operators: an
error where an input carries a derivative that the operators cannot give (a
custom op would drop a tangent and return a zero one), the ordinary result
where none does."""

from __future__ import annotations

import pytest

from conftest import pkg, submodule


def _operators(device):
    """{name: (function of one tensor, that tensor)}; other inputs are constants."""
    import torch

    M = pkg()
    bf16 = torch.bfloat16
    g = torch.Generator().manual_seed(0)

    def normal(*shape, dtype=bf16):
        return torch.randn(shape, generator=g).to(dtype).to(device)

    x, w, out = normal(4, 64), normal(64), normal(4, 64)
    gate, up, down = normal(32, 64), normal(32, 64), normal(64, 32)
    codes, scales, offsets = torch.full((8, 32), 37, dtype=torch.uint8, device=device), normal(8, 2), normal(8, 2)
    return {
        "rms_norm": (lambda a: M.rms_norm(a, w), x),
        "rms_norm by weight": (lambda a: M.rms_norm(x, a), w),
        "residual_norm": (lambda a: M.residual_norm(a, out, post_weight=w, next_weight=w)[1], x),
        "residual_norm by gate": (lambda a: M.residual_norm(x, out, gate=a)[0], normal(4, 1)),
        "residual_norm by expanded gate": (lambda a: M.residual_norm(x, out, gate=a)[0], normal(1, 1)),
        "gated_mlp": (lambda a: M.gated_mlp(a, gate, up, down, 2.0), x),
        "gated_mlp by down": (lambda a: M.gated_mlp(x, gate, up, a, 2.0), down),
        "int4_linear": (lambda a: M.int4_linear(a, codes, scales, offsets), x),
        "int4_linear by scales": (lambda a: M.int4_linear(x, codes, a, offsets), scales),
    }


NAMES = ["rms_norm", "rms_norm by weight", "residual_norm", "residual_norm by gate", "residual_norm by expanded gate",
         "gated_mlp", "gated_mlp by down", "int4_linear", "int4_linear by scales"]


def _refusals(fn, x):
    import torch

    fwd, t = torch.autograd.forward_ad, torch.ones_like(x)

    def dual():
        with fwd.dual_level():
            return fwd.unpack_dual(fn(fwd.make_dual(x, t)))

    def inner(a):  # the outer tangent within another function's jvp
        return torch.func.jvp(lambda b: fn(a).sum() + b, (t.sum(),), (t.sum(),))[1] + a.sum()

    calls = dict(
        dual=dual,
        jvp=lambda: torch.func.jvp(fn, (x,), (t,)),
        jvp_of_leaf=lambda: torch.func.jvp(fn, (x.clone().requires_grad_(),), (t,)),
        jacfwd=lambda: torch.func.jacfwd(fn)(x),
        nested=lambda: torch.func.jvp(inner, (x,), (t,)),
        jvp_of_vmap=lambda: torch.func.jvp(torch.func.vmap(fn), (x[None],), (t[None],)),
        vmap_of_jvp=lambda: torch.func.vmap(lambda v: torch.func.jvp(fn, (x,), (v,))[1])(t[None]),
        grad=lambda: torch.func.grad(lambda a: fn(a).float().sum())(x),
        vjp=lambda: torch.func.vjp(fn, x),
        compiled=lambda: torch.compile(lambda a, v: torch.func.jvp(fn, (a,), (v,))[1], backend="eager")(x, t),
    )
    for name, call in calls.items():
        with pytest.raises(RuntimeError, match="no derivative in forward mode"):
            call()
            pytest.fail(f"{name} was not refused")


@pytest.mark.parametrize("name", NAMES)
def test_derivatives_that_would_be_lost_are_refused(monkeypatch, name):
    """On the CPU: the refusal comes before any device work."""
    import torch

    monkeypatch.setattr(submodule("_native"), "same_device", lambda *a: 0)
    torch.compiler.reset()
    _refusals(*_operators("cpu")[name])


def test_the_mlp_in_4_bits_refuses_too(monkeypatch):
    import torch

    monkeypatch.setattr(submodule("_native"), "same_device", lambda *a: 0)
    M = pkg()
    mlp = M.Int4MLP.from_weights(torch.randn(32, 64), torch.randn(32, 64), torch.randn(64, 32), 2.0, group_size=32)
    with pytest.raises(RuntimeError, match="no derivative in forward mode"):
        torch.func.jvp(mlp, (torch.randn(4, 64).to(torch.bfloat16),), (torch.ones(4, 64, dtype=torch.bfloat16),))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_transforms_on_the_device(dev, name):
    import torch

    fn, x = _operators("cuda")[name]
    want = fn(x)
    torch.compiler.reset()
    _refusals(fn, x)
    # constants under a transform, made in it or not, and calls without a
    # tangent in a dual level are ordinary calls
    one = torch.ones((), device=dev)
    for constant in (lambda: x, lambda: x * 1, lambda: torch.func.vmap(lambda v: v * 1)(x)):
        y, t = torch.func.jvp(lambda b: b * fn(constant()).float(), (one,), (one,))
        assert torch.equal(y, want.float()) and torch.equal(t, want.float())
        d = torch.func.grad(lambda b: (b * fn(constant()).float()).sum())(one)
        assert torch.equal(d, want.float().sum())
    with torch.autograd.forward_ad.dual_level():
        assert torch.equal(fn(x), want)
    # vmap calls the op for every element
    xs = torch.stack([x, 2 * x, -x])
    assert torch.equal(torch.func.vmap(fn)(xs), torch.stack([fn(v) for v in xs]))
