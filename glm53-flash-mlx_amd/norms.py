"""Norms before and after a block, fused with its gate and residual scale.

The feed-forwards of this package take a normalised input and return what is
still to be added to the residual stream; ``rms_norm`` makes that input and
``residual_norm`` takes the result back:

    s            = out / rms(out) * post_weight       (no post_weight: s = out)
    new_residual = residual + scale * gate * s
    normed       = new_residual / rms(new_residual) * next_weight

with rms(v) = sqrt(mean(v^2) + eps) over the last axis.  Everything between
the loads and the stores is FP32 and each result is rounded once; ``normed``
is made of the new residual before it is rounded.  Both have gradients (first
order), and both are torch custom ops where a call is traced or transformed.
The reference takes its norms from mlx-vlm's layers and has no counterpart.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _native as N
from . import ops as _ops

_TYPES = (torch.bfloat16, torch.float32)
MAX_GATE_GROUPS = 512  # gate rows whose column sums are kept apart; more are expanded to one a token


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6, *,
             dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x / rms(x) * weight`` over the last axis, in ``dtype`` (x's own).

    x, weight and the result are bfloat16 or float32, each its own."""
    N.require_same_device(x, weight)
    dtype = x.dtype if dtype is None else dtype
    width = _check_rows("x", x)
    _check_weight("weight", weight, width)
    if dtype not in _TYPES:
        raise ValueError(f"rms_norm gives bfloat16 or float32, not {dtype}")
    form = (N.GATE_NONE, 1, 1.0, float(eps), True, dtype is torch.float32)
    return _call(x, None, None, None, weight, form)[1]


def residual_norm(residual: torch.Tensor, out: torch.Tensor, *, post_weight: torch.Tensor | None = None,
                  gate: torch.Tensor | None = None, scale: float = 1.0, next_weight: torch.Tensor | None = None,
                  eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor | None]:
    """A block's output taken into the residual stream: ``(new_residual,
    normed)`` as the module describes, ``normed`` None without `next_weight`.

    residual and out have one shape [..., width]; `new_residual` has
    residual's type, `normed` out's.  gate broadcasts against them: a value a
    channel ([width]), a token ([..., 1]), a sequence ([batch, 1, width]) or
    an element.  All tensors are bfloat16 or float32, each its own."""
    N.require_same_device(residual, out, post_weight, gate, next_weight)
    width = _check_rows("residual", residual)
    if out.shape != residual.shape:
        raise ValueError(f"out {tuple(out.shape)} must have residual's shape {tuple(residual.shape)}")
    _check_rows("out", out)
    _check_weight("post_weight", post_weight, width)
    _check_weight("next_weight", next_weight, width)
    kind, rows_per_gate = N.GATE_NONE, 1
    if gate is not None:
        gate, kind, rows_per_gate = _gate_form(gate, residual.shape)
    form = (kind, rows_per_gate, float(scale), float(eps), next_weight is not None, out.dtype is torch.float32)
    x, y = _call(residual, out, post_weight, gate, next_weight, form)
    return x, y if next_weight is not None else None


def _check_rows(name: str, t: torch.Tensor) -> int:
    if t.dtype not in _TYPES:
        raise ValueError(f"{name} must be bfloat16 or float32, got {t.dtype}")
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{name} must have a last axis of one element or more, got {tuple(t.shape)}")
    return t.shape[-1]


def _check_weight(name: str, t: torch.Tensor | None, width: int) -> None:
    if t is not None and (t.dtype not in _TYPES or t.dim() != 1 or t.shape[0] != width):
        raise ValueError(f"{name} must be a bfloat16 or float32 [{width}] tensor, got {tuple(t.shape)} {t.dtype}")


def _gate_form(gate: torch.Tensor, shape) -> tuple[torch.Tensor, int, int]:
    """The gate as the kernels take it, its kind, and the rows a gate row
    stands for.  Axes kept in front of axes of one element need no copy;
    other patterns, and more than MAX_GATE_GROUPS gate rows that each stand
    for several, are expanded, in float32 so that the gradient is summed
    before it is rounded."""
    if gate.dtype not in _TYPES:
        raise ValueError(f"gate must be bfloat16 or float32, got {gate.dtype}")
    width, rows = shape[-1], math.prod(shape[:-1])
    own = (1,) * (len(shape) - gate.dim()) + tuple(gate.shape)
    if len(own) != len(shape) or any(g != s and g != 1 for g, s in zip(own, shape)):
        raise ValueError(f"gate {tuple(gate.shape)} does not broadcast to {tuple(shape)}")
    lead, kept = own[:-1], 0
    while kept < len(lead) and lead[kept] == shape[kept]:
        kept += 1
    groups = math.prod(lead)
    prefix = all(g == 1 for g in lead[kept:])
    if own[-1] == width and rows > 0:
        if groups == rows:
            return gate, N.GATE_FULL, 1
        if prefix and groups <= MAX_GATE_GROUPS:
            return gate, N.GATE_COLUMNS, rows // groups
    elif own[-1] == 1 and groups == rows and rows > 0:
        return gate, N.GATE_ROWS, 1
    gate = gate.to(torch.float32).expand(*shape[:-1], own[-1])
    return gate, (N.GATE_FULL if own[-1] == width else N.GATE_ROWS), 1


def _call(residual, out, post_weight, gate, next_weight, form):
    tensors = (residual, out, post_weight, gate, next_weight)
    if _ops.direct(*tensors):
        return native_residual_norm(*tensors, *form, False)[:2]
    if _ops.eager(*tensors):
        return _ResidualNorm.apply(*tensors, form)
    return torch.ops.glm53.residual_norm(*tensors, *form)[:2]


def _ready(t: torch.Tensor | None) -> torch.Tensor | None:
    """Contiguous and, as far as its values' order needs it, 16-byte aligned."""
    if t is None:
        return None
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 and t.dim() and t.shape[-1] % 8 == 0 else t


def _mask(residual, out, post_weight, gate, next_weight, y_f32) -> int:
    m = N.NORM_F32_Y if y_f32 else 0
    for bit, t in ((N.NORM_F32_RESIDUAL, residual), (N.NORM_F32_OUT, out), (N.NORM_F32_POST, post_weight),
                   (N.NORM_F32_GATE, gate), (N.NORM_F32_NEXT, next_weight)):
        if t is not None and t.dtype is torch.float32:
            m |= bit
    return m


def _p(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def native_residual_norm(residual, out, post_weight, gate, next_weight, kind: int, rows_per_gate: int, scale: float,
                         eps: float, normed: bool, y_f32: bool, keep: bool = True):
    """The native call behind glm53::residual_norm: (new residual, or an empty
    tensor without out; normed, or an empty tensor; stats where kept)."""
    residual, out, gate = _ready(residual), _ready(out), _ready(gate)
    post_weight, next_weight = _ready(post_weight), _ready(next_weight)
    width = residual.shape[-1]
    rows = residual.numel() // width
    device = residual.device
    x = torch.empty_like(residual) if out is not None else residual.new_empty(0)
    y = torch.empty(residual.shape if normed else 0, dtype=torch.float32 if y_f32 else torch.bfloat16, device=device)
    stats = torch.empty((rows, 2) if keep else 0, dtype=torch.float32, device=device) if keep else None
    n = N.Norm(rows, width, rows_per_gate, residual.data_ptr(), _p(out), _p(post_weight), _p(gate), _p(next_weight),
               x.data_ptr() if out is not None else None, y.data_ptr() if normed else None, _p(stats), None, None, None,
               None, None, None, None, None, 0, kind, int(post_weight is not None),
               _mask(residual, out, post_weight, gate, next_weight, y_f32), scale, eps)
    if rows:
        N.run(device, N.lib().glm53_residual_norm, ctypes.byref(n))
    return x, y, stats


def native_residual_norm_backward(residual, out, post_weight, gate, next_weight, stats, d_new, d_y, kind: int,
                                  rows_per_gate: int, scale: float, eps: float, y_f32: bool, wanted: list[bool]):
    """The native call behind glm53::residual_norm_backward: the gradients of
    residual, out, post_weight, gate and next_weight that are `wanted`, empty
    tensors in place of the others."""
    inputs = [_ready(t) for t in (residual, out, post_weight, gate, next_weight)]
    residual, out, post_weight, gate, next_weight = inputs
    d_new, d_y = _ready(d_new), _ready(d_y)
    width = residual.shape[-1]
    rows = residual.numel() // width
    device = residual.device
    grads = [torch.empty_like(t) if t is not None and w else None for t, w in zip(inputs, wanted)]
    if rows == 0 or (d_new is None and d_y is None):
        return [residual.new_empty(0) if g is None else g.zero_() for g in grads]
    lib = N.lib()
    if d_y is None and grads[4] is not None:
        grads[4].zero_()
    gate_rows = rows // rows_per_gate if kind == N.GATE_COLUMNS else 1
    ws_bytes = lib.glm53_residual_norm_workspace_bytes(rows, width, gate_rows)
    ws = N.workspace(ws_bytes, device)
    n = N.Norm(rows, width, rows_per_gate, residual.data_ptr(), _p(out), _p(post_weight), _p(gate), _p(next_weight),
               None, None, stats.data_ptr(), _p(d_new), _p(d_y), _p(grads[0]), _p(grads[1]), _p(grads[2]), _p(grads[3]),
               _p(grads[4]) if d_y is not None else None, ws.data_ptr(), ws_bytes, kind, int(post_weight is not None),
               _mask(residual, out, post_weight, gate, next_weight, y_f32), scale, eps)
    N.run(device, lib.glm53_residual_norm_backward, ctypes.byref(n))
    return [residual.new_empty(0) if g is None else g for g in grads]


def _given(grads, wanted):
    return [g if w else None for g, w in zip(grads, wanted)]


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, out, post_weight, gate, next_weight, form):
        x, y, stats = native_residual_norm(residual, out, post_weight, gate, next_weight, *form)
        ctx.save_for_backward(residual, out, post_weight, gate, next_weight, stats)
        ctx.form = form
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*([x] if out is None else []), *([] if form[4] else [y]))
        return x, y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_new, d_y):
        saved = ctx.saved_tensors
        kind, rows_per_gate, scale, eps, normed, y_f32 = ctx.form
        wanted = [bool(w) for w in ctx.needs_input_grad[:5]]
        grads = native_residual_norm_backward(*saved, d_new if saved[1] is not None else None, d_y if normed else None,
                                              kind, rows_per_gate, scale, eps, y_f32, wanted)
        return (*_given(grads, wanted), None)
