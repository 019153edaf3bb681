"""Gated MLP in bf16 weights, trainable: what ``ClampedMLP`` is for frozen FP8
weights (patch.py:114-129 of the reference).

    G = x Wg^T, U = x Wu^T, h = silu(min(G, L)) * clip(U, -L, L), y = h Wd^T

Gate and up projections, activation and product are one kernel; sums, G, U
and the activation are FP32, h and y are rounded to bf16 once each (the FP8
path keeps the reference's rounding after every step instead).  A call that
may be differentiated keeps G and U in FP32, 8 bytes an intermediate value,
for the backward pass.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _native as N
from . import ops as _ops


def gated_mlp(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor, down_weight: torch.Tensor,
              limit: float | None = None) -> torch.Tensor:
    """``down(silu(min(gate(x), limit)) * clip(up(x), -limit, limit))``.

    x bfloat16 [..., hidden], gate_weight and up_weight bfloat16
    [intermediate, hidden], down_weight bfloat16 [hidden, intermediate], both
    widths multiples of 8; limit None: no clamp.  Differentiable (first order)
    in all four tensors."""
    N.require_same_device(x, gate_weight, up_weight, down_weight)
    weights = (gate_weight, up_weight, down_weight)
    for t in (x, *weights):
        if t.dtype != torch.bfloat16:
            raise ValueError(f"the gated MLP takes bfloat16 tensors, got {t.dtype}")
    if any(w.dim() != 2 for w in weights) or x.dim() < 1:
        raise ValueError("the gated MLP takes x [..., hidden] and 2-D weights")
    inter, hidden = gate_weight.shape
    if up_weight.shape != (inter, hidden) or down_weight.shape != (hidden, inter) or x.shape[-1] != hidden:
        raise ValueError(f"shapes do not match: x {tuple(x.shape)}, gate {tuple(gate_weight.shape)}, "
                         f"up {tuple(up_weight.shape)}, down {tuple(down_weight.shape)}")
    if hidden % 8 or inter % 8 or hidden == 0 or inter == 0:
        raise ValueError(f"hidden {hidden} and intermediate {inter} must be multiples of 8")
    limit = math.inf if limit is None else float(limit)
    if not limit > 0:
        raise ValueError(f"limit must be positive, got {limit}")
    if _ops.direct(x, *weights):
        return native_gated_mlp(x, *weights, limit, False)[0]
    if _ops.eager(x, *weights):
        return _GatedMLP.apply(x, *weights, limit)
    keep = torch.is_grad_enabled() and any(t.requires_grad for t in (x, *weights))
    return torch.ops.glm53.gated_mlp(x, *weights, limit, keep)[0]


def _ready(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and 16-byte aligned."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def native_gated_mlp(x, gate_weight, up_weight, down_weight, limit: float, keep: bool):
    """The native call behind glm53::gated_mlp: y, and G and U where kept
    (empty tensors otherwise)."""
    x, gate_weight, up_weight, down_weight = _ready(x), _ready(gate_weight), _ready(up_weight), _ready(down_weight)
    inter, hidden = gate_weight.shape
    rows = x.numel() // hidden
    y = torch.empty_like(x)
    gate = torch.empty((rows, inter) if keep else 0, dtype=torch.float32, device=x.device)
    up = torch.empty_like(gate)
    if rows:
        lib = N.lib()
        ws_bytes = lib.glm53_gated_mlp_workspace_bytes(rows, hidden, inter)
        ws = N.workspace(ws_bytes, x.device)
        d = N.GatedMLP(rows, hidden, inter, x.data_ptr(), gate_weight.data_ptr(), up_weight.data_ptr(),
                       down_weight.data_ptr(), y.data_ptr(), gate.data_ptr() if keep else None,
                       up.data_ptr() if keep else None, None, None, None, None, None, ws.data_ptr(), ws_bytes,
                       limit)
        N.run(x.device, lib.glm53_gated_mlp, ctypes.byref(d))
    return y, gate, up


def native_gated_mlp_backward(x, gate_weight, up_weight, down_weight, gate, up, d_y, limit: float, wanted: list[bool]):
    """The native call behind glm53::gated_mlp_backward: the gradients of x
    and the weights that are `wanted`, empty tensors in place of the others."""
    inputs = [_ready(t) for t in (x, gate_weight, up_weight, down_weight)]
    d_y = _ready(d_y)
    inter, hidden = gate_weight.shape
    rows = x.numel() // hidden
    grads = [torch.empty_like(t) if w else None for t, w in zip(inputs, wanted)]
    if rows == 0:
        return [x.new_empty(0) if g is None else g.zero_() for g in grads]
    lib = N.lib()
    ws_bytes = lib.glm53_gated_mlp_backward_workspace_bytes(rows, hidden, inter)
    ws = N.workspace(ws_bytes, x.device)
    d = N.GatedMLP(rows, hidden, inter, *(t.data_ptr() for t in inputs), None, gate.data_ptr(), up.data_ptr(),
                   d_y.data_ptr(), *(None if g is None else g.data_ptr() for g in grads), ws.data_ptr(), ws_bytes, limit)
    N.run(x.device, lib.glm53_gated_mlp_backward, ctypes.byref(d))
    return [x.new_empty(0) if g is None else g for g in grads]


class _GatedMLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_weight, up_weight, down_weight, limit):
        y, gate, up = native_gated_mlp(x, gate_weight, up_weight, down_weight, limit, True)
        ctx.save_for_backward(x, gate_weight, up_weight, down_weight, gate, up)
        ctx.limit = limit
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y):
        wanted = [bool(w) for w in ctx.needs_input_grad[:4]]
        grads = native_gated_mlp_backward(*ctx.saved_tensors, d_y, ctx.limit, wanted)
        return (*(g if w else None for g, w in zip(grads, wanted)), None)


class GatedMLP(torch.nn.Module):
    """``gated_mlp`` with its weights as parameters, named as ClampedMLP's projections."""

    def __init__(self, hidden_size: int, intermediate_size: int, limit: float | None = None, device=None):
        super().__init__()
        self.gate_proj = torch.nn.Linear(hidden_size, intermediate_size, bias=False, device=device, dtype=torch.bfloat16)
        self.up_proj = torch.nn.Linear(hidden_size, intermediate_size, bias=False, device=device, dtype=torch.bfloat16)
        self.down_proj = torch.nn.Linear(intermediate_size, hidden_size, bias=False, device=device, dtype=torch.bfloat16)
        self.limit = limit

    def forward(self, x):
        return gated_mlp(x, self.gate_proj.weight, self.up_proj.weight, self.down_proj.weight, self.limit)

    def to_int4(self, group_size: int = 64, symmetric: bool = False):
        """The served form: an Int4MLP of these weights."""
        from .int4 import Int4MLP

        return Int4MLP.from_weights(self.gate_proj.weight, self.up_proj.weight, self.down_proj.weight, self.limit,
                                    group_size=group_size, symmetric=symmetric)
