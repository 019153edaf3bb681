"""CPU checks of the dense feed-forward block's C entry points: arguments are
refused before any device work (status 1 with a message), sizes of
workspaces, and no CPU fallback in the Python functions."""

from __future__ import annotations

import ctypes

import pytest

from conftest import pkg, submodule

FAKE = 1 << 20  # never dereferenced: every call here is refused or has nothing to do


@pytest.fixture(scope="module")
def N():
    return submodule("_native")


@pytest.fixture(scope="module")
def libso(N):
    return N.load_library()


def _norm(N, **changes):
    n = N.Norm(rows=4, width=64, rows_per_gate=4, residual=FAKE, out=FAKE, post_weight=FAKE, gate=FAKE, next_weight=FAKE,
               new_residual=FAKE, y=FAKE, stats=FAKE, gate_kind=N.GATE_COLUMNS, post_norm=1, scale=1.0, eps=1e-6)
    for name, value in changes.items():
        setattr(n, name, value)
    return ctypes.byref(n)


@pytest.mark.parametrize("changes, message", [
    (dict(rows=-1), "invalid shape"), (dict(width=0), "invalid shape"), (dict(rows=1 << 31), "invalid shape"),
    (dict(width=16385), "exceeds"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(f32_mask=64), "f32_mask"),
    (dict(gate_kind=4), "gate kind"), (dict(gate=None), "gate"), (dict(gate_kind=0), "gate"),
    (dict(rows_per_gate=0), "rows_per_gate"), (dict(rows_per_gate=3), "rows_per_gate"),
    (dict(out=None), "without a block output"), (dict(post_norm=0), "post_weight"),
    (dict(residual=None), "null"), (dict(new_residual=None), "null"),
    # rows of another type over rows that are still to be read
    (dict(new_residual=FAKE, f32_mask=1), "type"), (dict(y=FAKE, f32_mask=32, new_residual=2 * FAKE), "type"),
    (dict(out=None, gate=None, gate_kind=0, post_weight=None, post_norm=0, f32_mask=1), "type"),
    (dict(out=None, gate=None, gate_kind=0, post_weight=None, post_norm=0, y=None), "nothing to compute"),
])
def test_norm_refusals(N, libso, changes, message):
    assert libso.glm53_residual_norm(_norm(N, **changes), None) == N.INVALID_ARGUMENT
    assert message in libso.glm53_last_error().decode()


@pytest.mark.parametrize("changes, message", [
    (dict(), "workspace"), (dict(workspace=FAKE, workspace_bytes=16), "workspace"),
    (dict(workspace=FAKE + 4, workspace_bytes=1 << 30), "workspace"), (dict(stats=None), "null"),
    (dict(gate=None, gate_kind=0, d_gate=FAKE), "d_gate"),
    (dict(post_norm=0, post_weight=None, d_post_weight=FAKE), "d_post_weight"),
    (dict(out=None, gate=None, gate_kind=0, post_weight=None, post_norm=0, d_out=FAKE), "d_out"),
])
def test_norm_backward_refusals(N, libso, changes, message):
    assert libso.glm53_residual_norm_backward(_norm(N, **changes), None) == N.INVALID_ARGUMENT
    assert message in libso.glm53_last_error().decode()


def test_norm_without_rows_and_workspace_sizes(N, libso):
    assert libso.glm53_residual_norm(None, None) == N.INVALID_ARGUMENT
    assert libso.glm53_residual_norm(_norm(N, rows=0, residual=None), None) == N.OK
    size = libso.glm53_residual_norm_workspace_bytes
    assert size(0, 64, 1) == size(4, 0, 1) == size(4, 64, 5) == size(4, 64, 0) == 0
    assert size(4, 64, 1) == 4 * 3 * 64 * 4
    assert size(8192, 4096, 1) <= 512 * 3 * 4096 * 4
    assert size(8192, 64, 8192) == 8192 * 3 * 64 * 4


def _gated(N, **changes):
    d = N.GatedMLP(rows=4, hidden=64, intermediate=32, x=FAKE, gate_weight=FAKE, up_weight=FAKE, down_weight=FAKE, y=FAKE,
                   gate=FAKE, up=FAKE, h=FAKE, d_y=FAKE, workspace=FAKE, workspace_bytes=1 << 30, limit=1.0)
    for name, value in changes.items():
        setattr(d, name, value)
    return ctypes.byref(d)


@pytest.mark.parametrize("changes, message", [
    (dict(rows=-1), "invalid shape"), (dict(rows=1 << 31), "invalid shape"), (dict(hidden=0), "invalid shape"),
    (dict(intermediate=0), "invalid shape"), (dict(hidden=60), "multiples of 8"), (dict(intermediate=4), "multiples of 8"),
    (dict(hidden=1 << 23), "widths"), (dict(limit=0.0), "limit"), (dict(limit=-1.0), "limit"),
    (dict(limit=float("nan")), "limit"), (dict(x=FAKE + 2), "aligned"), (dict(down_weight=FAKE + 8), "aligned"),
    (dict(up=None), "together"), (dict(h=None), "together"), (dict(x=None), "null"), (dict(gate_weight=None), "null"),
    (dict(workspace=None), "workspace"), (dict(workspace=FAKE + 16), "workspace"), (dict(workspace_bytes=8), "workspace"),
])
def test_gated_refusals(N, libso, changes, message):
    for entry in (libso.glm53_gated_mlp, libso.glm53_gated_mlp_backward):
        assert entry(_gated(N, **changes), None) == N.INVALID_ARGUMENT
        assert message in libso.glm53_last_error().decode()


def test_gated_empty_calls_and_workspace_sizes(N, libso):
    assert libso.glm53_gated_mlp(None, None) == N.INVALID_ARGUMENT
    assert libso.glm53_gated_mlp(_gated(N, rows=0, x=None), None) == N.OK
    assert libso.glm53_gated_mlp(_gated(N, y=None), None) == N.INVALID_ARGUMENT
    assert libso.glm53_gated_mlp_backward(_gated(N, rows=0), None) == N.INVALID_ARGUMENT
    assert libso.glm53_gated_mlp_backward(_gated(N, gate=None, up=None, h=None), None) == N.INVALID_ARGUMENT
    for size in (libso.glm53_gated_mlp_workspace_bytes, libso.glm53_gated_mlp_backward_workspace_bytes):
        assert size(0, 64, 32) == size(4, 0, 32) == size(4, 64, 0) == 0
        assert size(4, 64, 32) >= 4 * 32 * 2


def _int4(N, **changes):
    w = N.Int4Weight(codes=FAKE, scales=FAKE, offsets=FAKE, bias=FAKE, out_features=48, in_features=128, group=64)
    for name, value in changes.items():
        setattr(w, name, value)
    return ctypes.byref(w)


@pytest.mark.parametrize("changes, message", [
    (dict(out_features=0), "invalid shape"), (dict(in_features=0), "invalid shape"), (dict(group=16), "group"),
    (dict(group=0), "group"), (dict(in_features=96), "multiple of the group"), (dict(codes=None), "null"),
    (dict(scales=None), "null"), (dict(codes=FAKE + 8), "aligned"), (dict(in_features=1 << 23), "too large"),
    (dict(out_features=(1 << 22) + 1), "too large"),
])
def test_int4_refusals(N, libso, changes, message):
    assert libso.glm53_int4_linear(_int4(N, **changes), FAKE, 4, FAKE, FAKE, 1 << 30, None) == N.INVALID_ARGUMENT
    assert message in libso.glm53_last_error().decode()


def test_int4_refuses_call_arguments(N, libso):
    for x, rows, y in ((FAKE, -1, FAKE), (FAKE, 1 << 31, FAKE), (None, 4, FAKE), (FAKE, 4, None), (FAKE + 2, 4, FAKE),
                       (FAKE, 4, FAKE + 8)):
        assert libso.glm53_int4_linear(_int4(N), x, rows, y, FAKE, 1 << 30, None) == N.INVALID_ARGUMENT
    assert libso.glm53_int4_linear(None, FAKE, 4, FAKE, None, 0, None) == N.INVALID_ARGUMENT
    assert libso.glm53_int4_linear(_int4(N), None, 0, None, None, 0, None) == N.OK
    size = libso.glm53_int4_linear_workspace_bytes
    assert size(0, 48, 128) == size(4, 0, 128) == size(4, 48, 0) == 0


def test_quantize_int4_gives_the_nearest_codes():
    """Codes, scales and offsets made on the CPU: nearest codes for the rounded
    tables, constant and zero groups, and refusals."""
    import torch

    M = pkg()
    g = torch.Generator()
    g.manual_seed(0)
    w = torch.randn(6, 128, generator=g)
    w[0, :64], w[1, 64:] = 0.0, 0.75
    for symmetric in (False, True):
        for dtype in (torch.bfloat16, torch.float32):
            codes, scales, offsets = M.quantize_int4(w, 64, symmetric, dtype)
            assert codes.shape == (6, 64) and scales.shape == (6, 2) and scales.dtype == dtype
            q = torch.stack([codes & 15, codes >> 4], 2).view(6, 2, 64).double()
            s = scales.double()[:, :, None]
            o = -8 * s if symmetric else offsets.double()[:, :, None]
            v = w.double().view(6, 2, 64)
            every = s[..., None] * torch.arange(16) + o[..., None]  # [6, 2, 1, 16]
            best = (every - v[..., None]).abs().amin(3)
            assert ((q * s + o - v).abs() <= best + 1e-6).all()
            assert ((q * s + o)[0, 0] == 0).all()
    for bad in (lambda: M.quantize_int4(w, 48), lambda: M.quantize_int4(w[:, :96], 64), lambda: M.quantize_int4(w[0], 64),
                lambda: M.quantize_int4(w.int(), 64), lambda: M.quantize_int4(w, 64, dtype=torch.float16),
                lambda: M.quantize_int4(w / 0, 64), lambda: M.quantize_int4(w.sign() * 3e38, 64),
                lambda: M.quantize_int4(w.sign() * 3.4e38, 64, True), lambda: M.Int4Linear(96, 8, group_size=64),
                lambda: M.Int4MLP(M.Int4Linear(64, 64), M.Int4Linear(64, 64)),
                lambda: M.Int4MLP.from_weights(w, w[:3], w.t())):
        with pytest.raises(ValueError):
            bad()


def test_struct_layouts(N, tmp_path):
    """Sizes and offsets of the block's structs in the header, compiled as C,
    are those of the Python binding."""
    import subprocess

    from conftest import ROOT

    structs = {"glm53_norm": N.Norm, "glm53_gated_mlp_desc": N.GatedMLP, "glm53_int4_weight": N.Int4Weight}
    lines = ["#include <glm53_moe.h>", "#include <stdio.h>", "int main(void) {"]
    want = {}
    for name, py in structs.items():
        lines.append(f'  printf("{name} %zu\\n", sizeof({name}));')
        want[name] = ctypes.sizeof(py)
        for field, _ in py._fields_:
            lines.append(f'  printf("{name}.{field} %zu\\n", offsetof({name}, {field}));')
            want[f"{name}.{field}"] = getattr(py, field).offset
    (tmp_path / "s.c").write_text("\n".join([*lines, "  return 0;", "}"]))
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    out = subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout
    assert {a: int(b) for a, b in (line.split() for line in out.splitlines())} == want


def test_python_functions_refuse_cpu_tensors():
    import torch

    M = pkg()
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.ones(64)
    for call in (lambda: M.rms_norm(x, w), lambda: M.residual_norm(x, x, next_weight=w),
                 lambda: M.gated_mlp(x, x, x, x.t()),
                 lambda: M.int4_linear(x, torch.zeros(8, 32, dtype=torch.uint8), torch.ones(8, 1))):
        with pytest.raises((RuntimeError, ValueError)):
            call()


@pytest.mark.parametrize("limit", [0.0, -1.0, float("nan")])
def test_the_mlp_in_4_bits_refuses_the_limits_that_gated_mlp_refuses(limit):
    import torch

    M = pkg()
    mlp = M.Int4MLP.from_weights(torch.randn(32, 64), torch.randn(32, 64), torch.randn(64, 32), limit, group_size=32)
    with pytest.raises(ValueError, match="limit must be positive"):
        mlp(torch.zeros(2, 64, dtype=torch.bfloat16))
