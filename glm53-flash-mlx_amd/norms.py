"""Norms before and after a block, fused with its gate and residual scale.

The feed-forwards of this package take a normalised input and return what is
still to be added to the residual stream; ``rms_norm`` makes that input and
``residual_norm`` takes the result back:

    s            = out / rms(out) * post_weight       (no post_weight: s = out)
    new_residual = residual + scale * gate * s
    normed       = new_residual / rms(new_residual) * next_weight

with rms(v) = sqrt(mean(v^2) + eps) over the last axis.  Everything between
the loads and the stores is FP32 and each result is rounded once; ``normed``
is made of the new residual before it is rounded.  Squares are FP32 too: rows of
values past 2^63 have an infinite rms, and norm to 0.  Both have gradients (first
order, in reverse mode; forward mode and torch.func's grad, vjp and jvp raise),
and both are torch custom ops where a call is traced.
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
    N.same_device(x, weight)
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
    N.same_device(residual, out, post_weight, gate, next_weight)
    width = _check_rows("residual", residual)
    shape = residual.shape
    if out.shape != shape:
        raise ValueError(f"out {tuple(out.shape)} must have residual's shape {tuple(shape)}")
    if out.dtype not in _TYPES:
        raise ValueError(f"out must be bfloat16 or float32, got {out.dtype}")
    _check_weight("post_weight", post_weight, width)
    _check_weight("next_weight", next_weight, width)
    kind, rows_per_gate = N.GATE_NONE, 1
    if gate is not None:
        gate, kind, rows_per_gate = _gate_form(gate, shape)
    form = (kind, rows_per_gate, float(scale), float(eps), next_weight is not None, out.dtype is torch.float32)
    x, y = _call(residual, out, post_weight, gate, next_weight, form)
    return x, y if next_weight is not None else None


def _check_rows(name: str, t: torch.Tensor) -> int:
    if t.dtype not in _TYPES:
        raise ValueError(f"{name} must be bfloat16 or float32, got {t.dtype}")
    shape = t.shape
    if not shape or shape[-1] < 1:
        raise ValueError(f"{name} must have a last axis of one element or more, got {tuple(shape)}")
    return shape[-1]


def _check_weight(name: str, t: torch.Tensor | None, width: int) -> None:
    if t is not None and (t.dtype not in _TYPES or t.shape != (width,)):
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
    if gate.shape == (width,) and rows > 0:  # a value a channel
        return gate, N.GATE_COLUMNS, rows
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
        x, y, _ = native_residual_norm(*tensors, *form, False)
        return x, y
    if _ops.eager(*tensors):
        return _ResidualNorm.apply(*tensors, form)
    _ops.refuse_transforms("rms_norm" if out is None else "residual_norm", *tensors)
    return torch.ops.glm53.residual_norm(*tensors, *form)[:2]


def _taken(t: torch.Tensor | None):
    """(t as the kernels take it, its address); (None, None) where absent."""
    if t is None:
        return None, None
    if not t.is_contiguous():
        t = t.contiguous()
    return t, t.data_ptr()


def _f32(t: torch.Tensor | None, bit: int) -> int:
    return bit if t is not None and t.dtype is torch.float32 else 0


def _mask(residual, out, post_weight, gate, next_weight, y_f32) -> int:
    return (_f32(residual, N.NORM_F32_RESIDUAL) | _f32(out, N.NORM_F32_OUT) | _f32(post_weight, N.NORM_F32_POST)
            | _f32(gate, N.NORM_F32_GATE) | _f32(next_weight, N.NORM_F32_NEXT) | (N.NORM_F32_Y if y_f32 else 0))


def native_residual_norm(residual, out, post_weight, gate, next_weight, kind: int, rows_per_gate: int, scale: float,
                         eps: float, normed: bool, y_f32: bool, keep: bool = True):
    """The native call behind glm53::residual_norm: (new residual, normed, stats),
    None for what is not made."""
    residual, p_residual = _taken(residual)
    out, p_out = _taken(out)
    post_weight, p_post = _taken(post_weight)
    gate, p_gate = _taken(gate)
    next_weight, p_next = _taken(next_weight)
    shape = residual.shape
    width = shape[-1]
    rows = residual.numel() // width
    x = p_x = y = p_y = stats = p_stats = None
    if out is not None:
        x = torch.empty_like(residual)
        p_x = x.data_ptr()
    if normed:
        if y_f32 == (residual.dtype is torch.float32):
            y = torch.empty_like(residual)
        else:
            y = residual.new_empty(shape, dtype=torch.float32 if y_f32 else torch.bfloat16)
        p_y = y.data_ptr()
    if keep:
        stats = residual.new_empty((rows, 2), dtype=torch.float32)
        p_stats = stats.data_ptr()
    if rows:
        n = N.Norm(rows, width, rows_per_gate, p_residual, p_out, p_post, p_gate, p_next, p_x, p_y, p_stats, None, None,
                   None, None, None, None, None, None, 0, kind, post_weight is not None,
                   _mask(residual, out, post_weight, gate, next_weight, y_f32), scale, eps)
        N.run(residual.get_device(), N.lib().glm53_residual_norm, ctypes.byref(n))
    return x, y, stats


def native_residual_norm_backward(residual, out, post_weight, gate, next_weight, stats, d_new, d_y, kind: int,
                                  rows_per_gate: int, scale: float, eps: float, y_f32: bool, wanted: list[bool]):
    """The native call behind glm53::residual_norm_backward: the gradients of
    residual, out, post_weight, gate and next_weight that are `wanted`, None in
    place of the others."""
    (residual, out, post_weight, gate, next_weight), addresses = zip(*map(_taken, (residual, out, post_weight, gate,
                                                                                   next_weight)))
    d_new, p_new = _taken(d_new)
    d_y, p_y = _taken(d_y)
    width = residual.shape[-1]
    rows = residual.numel() // width
    grads = [torch.empty_like(t) if t is not None and w else None
             for t, w in zip((residual, out, post_weight, gate, next_weight), wanted)]
    if rows == 0 or (d_new is None and d_y is None):
        return [None if g is None else g.zero_() for g in grads]
    lib = N.lib()
    p_grads = [None if g is None else g.data_ptr() for g in grads]
    if d_y is None and grads[4] is not None:
        grads[4].zero_()
        p_grads[4] = None
    gate_rows = rows // rows_per_gate if kind == N.GATE_COLUMNS else 1
    ws_bytes = lib.glm53_residual_norm_workspace_bytes(rows, width, gate_rows)
    ws = residual.new_empty(ws_bytes, dtype=torch.uint8)
    n = N.Norm(rows, width, rows_per_gate, *addresses, None, None, stats.data_ptr(), p_new, p_y, *p_grads, ws.data_ptr(),
               ws_bytes, kind, post_weight is not None, _mask(residual, out, post_weight, gate, next_weight, y_f32),
               scale, eps)
    N.run(residual.get_device(), lib.glm53_residual_norm_backward, ctypes.byref(n))
    return grads


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, out, post_weight, gate, next_weight, form):
        x, y, stats = native_residual_norm(residual, out, post_weight, gate, next_weight, *form)
        ctx.save_for_backward(residual, out, post_weight, gate, next_weight, stats)
        ctx.form = form
        ctx.set_materialize_grads(False)
        return x, y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_new, d_y):
        kind, rows_per_gate, scale, eps, _, y_f32 = ctx.form
        return (*native_residual_norm_backward(*ctx.saved_tensors, d_new, d_y, kind, rows_per_gate, scale, eps, y_f32,
                                               ctx.needs_input_grad), None)
