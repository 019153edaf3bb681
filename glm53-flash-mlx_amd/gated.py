"""Gated MLP in bf16 weights, trainable: what ``ClampedMLP`` is for frozen FP8
weights (patch.py:114-129 of the reference).

    G = x Wg^T, U = x Wu^T, h = silu(min(G, L)) * clip(U, -L, L), y = h Wd^T

Gate and up projections, activation and product are one kernel; sums, G, U
and the activation are FP32, h and y are rounded to bf16 once each (the FP8
path keeps the reference's rounding after every step instead).  Over few rows,
16, or 32 of at most 4,096 hidden and 2,048 intermediate columns, h enters the
down projection in two bf16 parts, 16 bits, so a token's result beside few
others differs from its result in a batch by that rounding (2^-8 of h at most);
so do dG, dU and h in the gradients, up to 16 rows.  A call that
may be differentiated keeps G and U in FP32 and h, 10 bytes an intermediate
value, for the backward pass.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _native as N
from . import ops as _ops


FEW_ROWS = 16  # up to here what is rounded as an operand is carried in two bf16 parts


def gated_mlp(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor, down_weight: torch.Tensor,
              limit: float | None = None) -> torch.Tensor:
    """``down(silu(min(gate(x), limit)) * clip(up(x), -limit, limit))``.

    x bfloat16 [..., hidden], gate_weight and up_weight bfloat16
    [intermediate, hidden], down_weight bfloat16 [hidden, intermediate], both
    widths multiples of 8; limit None: no clamp.  Differentiable (first order, in
    reverse mode; forward mode and torch.func's grad, vjp and jvp raise) in all
    four tensors."""
    N.same_device(x, gate_weight, up_weight, down_weight)
    weights = (gate_weight, up_weight, down_weight)
    x_shape, shape = x.shape, gate_weight.shape
    bf16 = torch.bfloat16
    if x.dtype is not bf16 or gate_weight.dtype is not bf16 or up_weight.dtype is not bf16 or down_weight.dtype is not bf16:
        raise ValueError(f"the gated MLP takes bfloat16 tensors, got {[t.dtype for t in (x, *weights)]}")
    if len(shape) != 2 or not x_shape:
        raise ValueError("the gated MLP takes x [..., hidden] and 2-D weights")
    inter, hidden = shape
    if up_weight.shape != shape or down_weight.shape != (hidden, inter) or x_shape[-1] != hidden:
        raise ValueError(f"shapes do not match: x {tuple(x_shape)}, gate {tuple(shape)}, "
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
    _ops.refuse_transforms("gated_mlp", x, *weights)
    keep = torch.is_grad_enabled() and any(t.requires_grad for t in (x, *weights))
    return torch.ops.glm53.gated_mlp(x, *weights, limit, keep)[0]


def native_gated_mlp(x, gate_weight, up_weight, down_weight, limit: float, keep: bool):
    """The native call behind glm53::gated_mlp: y, and G, U and h where kept."""
    x, gate_weight, up_weight, down_weight = map(N.operand, (x, gate_weight, up_weight, down_weight))
    inter, hidden = gate_weight.shape
    rows = x.numel() // hidden
    y = torch.empty_like(x)
    gate = up = h = p_gate = p_up = p_h = None
    if keep:
        gate = x.new_empty((rows, inter), dtype=torch.float32)
        up = torch.empty_like(gate)
        h = x.new_empty((2, rows, inter) if rows <= FEW_ROWS else (rows, inter))
        p_gate, p_up, p_h = gate.data_ptr(), up.data_ptr(), h.data_ptr()
    if rows:
        lib = N.lib()
        ws_bytes = lib.glm53_gated_mlp_workspace_bytes(rows, hidden, inter)
        ws = N.workspace(ws_bytes, x.device)
        d = N.GatedMLP(rows, hidden, inter, x.data_ptr(), gate_weight.data_ptr(), up_weight.data_ptr(),
                       down_weight.data_ptr(), y.data_ptr(), p_gate, p_up, p_h, None, None, None, None, None, ws.data_ptr(),
                       ws_bytes, limit)
        N.run(x.get_device(), lib.glm53_gated_mlp, ctypes.byref(d))
    return y, gate, up, h


def native_gated_mlp_backward(x, gate_weight, up_weight, down_weight, gate, up, h, d_y, limit: float, wanted: list[bool]):
    """The native call behind glm53::gated_mlp_backward: the gradients of x
    and the weights that are `wanted`, None in place of the others."""
    inputs = [N.operand(t) for t in (x, gate_weight, up_weight, down_weight)]
    d_y = N.operand(d_y)
    inter, hidden = gate_weight.shape
    rows = x.numel() // hidden
    grads = [torch.empty_like(t) if w else None for t, w in zip(inputs, wanted)]
    if rows == 0:
        return [None if g is None else g.zero_() for g in grads]
    lib = N.lib()
    ws_bytes = lib.glm53_gated_mlp_backward_workspace_bytes(rows, hidden, inter)
    ws = N.workspace(ws_bytes, x.device)
    d = N.GatedMLP(rows, hidden, inter, *(t.data_ptr() for t in inputs), None, gate.data_ptr(), up.data_ptr(),
                   h.data_ptr(), d_y.data_ptr(), *(None if g is None else g.data_ptr() for g in grads), ws.data_ptr(), ws_bytes, limit)
    N.run(x.get_device(), lib.glm53_gated_mlp_backward, ctypes.byref(d))
    return grads


class _GatedMLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_weight, up_weight, down_weight, limit):
        y, *kept = native_gated_mlp(x, gate_weight, up_weight, down_weight, limit, True)
        ctx.save_for_backward(x, gate_weight, up_weight, down_weight, *kept)
        ctx.limit = limit
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y):
        return (*native_gated_mlp_backward(*ctx.saved_tensors, d_y, ctx.limit, ctx.needs_input_grad), None)


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
