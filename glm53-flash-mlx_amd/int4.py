"""Linear layers with 4-bit weights and group scales.

W[n, k] = scales[n, k / g] * q[n, k] + offsets[n, k / g], q in 0..15, one
scale and offset for g = 32, 64 or 128 columns of a row: half the bytes of the
block-FP8 weights, which is what a call over few tokens costs.  Codes lie two
to a byte, the even column in the low half.  No gradients: the served form of
trained weights (``GatedMLP.to_int4``).  The reference's weights are FP8 and
have no counterpart.

A product multiplies by the codes and scales the sums of each group in FP32,
whatever the number of rows: the weights are those that codes and tables
define, not their roundings to bf16, in decode and in prefill alike.  Above 128
rows a call writes the codes' bf16 values into a workspace of 2.25 bytes a
weight and more (4096 x 4096: 38 MB), which torch's allocator keeps for the next
one.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _native as N
from . import ops as _ops

GROUP_SIZES = (32, 64, 128)
FEW_ROWS = 32  # up to here no call takes a workspace


def int4_linear(x: torch.Tensor, weight: torch.Tensor, scales: torch.Tensor, offsets: torch.Tensor | None = None,
                bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ W.T + bias`` with W as the module describes.

    x bfloat16 [..., in]; weight uint8 [out, in / 2]; scales and offsets [out,
    in / g], bias [out], all bfloat16 or all float32; offsets None: -8 scales.
    FP32 sums, rounded once; no weight is rounded."""
    N.same_device(x, weight, scales, offsets, bias)
    x_shape, w_shape, s_shape, table = x.shape, weight.shape, scales.shape, scales.dtype
    if x.dtype is not torch.bfloat16:
        raise ValueError(f"activations must be bfloat16, got {x.dtype}")
    if weight.dtype is not torch.uint8 or len(w_shape) != 2:
        raise ValueError(f"expected 2-D uint8 codes, got {tuple(w_shape)} {weight.dtype}")
    out_features, in_features = w_shape[0], 2 * w_shape[1]
    if not x_shape or x_shape[-1] != in_features:
        raise ValueError(f"input {tuple(x_shape)} does not end in the weight's width {in_features}")
    if (table is not torch.bfloat16 and table is not torch.float32) or len(s_shape) != 2 or s_shape[0] != out_features:
        raise ValueError(f"scales must be bfloat16 or float32 [{out_features}, groups], got {tuple(s_shape)} {table}")
    groups = s_shape[1]
    if out_features == 0 or groups == 0 or in_features not in (32 * groups, 64 * groups, 128 * groups):
        raise ValueError(f"{groups} groups over {in_features} columns: groups hold {GROUP_SIZES} columns")
    if offsets is not None and (offsets.shape != s_shape or offsets.dtype is not table):
        raise ValueError(f"offsets must match scales, got {tuple(offsets.shape)} {offsets.dtype}")
    if bias is not None and (bias.shape != (out_features,) or bias.dtype is not table):
        raise ValueError(f"bias must be {table} [{out_features}], got {tuple(bias.shape)} {bias.dtype}")
    if _ops.direct(x, weight, scales, offsets, bias):
        return native_int4_linear(x, weight, scales, offsets, bias)
    _ops.refuse_transforms("int4_linear", x, scales, offsets, bias)
    return torch.ops.glm53.int4_linear(x, weight, scales, offsets, bias)


def native_int4_linear(x, weight, scales, offsets, bias):
    """The native call behind glm53::int4_linear (arguments validated)."""
    out_features, half = weight.shape
    in_features = 2 * half
    x, weight, scales = N.operand(x), N.operand(weight), scales.contiguous()
    if offsets is not None:
        offsets = offsets.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    rows = x.numel() // in_features
    y = x.new_empty((rows, out_features) if x.dim() == 2 else (*x.shape[:-1], out_features))
    if rows == 0:
        return y
    lib = N.lib()
    ws, ws_bytes = None, 0
    if rows > FEW_ROWS:
        ws_bytes = lib.glm53_int4_linear_workspace_bytes(rows, out_features, in_features)
        ws = N.workspace(ws_bytes, x.device)
    w = N.Int4Weight(weight.data_ptr(), scales.data_ptr(), None if offsets is None else offsets.data_ptr(),
                     None if bias is None else bias.data_ptr(), out_features, in_features,
                     in_features // scales.shape[1], scales.dtype is torch.float32)
    N.run(x.get_device(), lib.glm53_int4_linear, ctypes.byref(w), x.data_ptr(), rows, y.data_ptr(),
          None if ws is None else ws.data_ptr(), ws_bytes)
    return y


def quantize_int4(weight: torch.Tensor, group_size: int = 64, symmetric: bool = False,
                  dtype: torch.dtype = torch.bfloat16):
    """``(codes, scales, offsets)`` of a [out, in] weight: per row and group
    the codes nearest to it between its least and largest value, or
    (symmetric, offsets None) between -8 and 7 scales.  Scales and offsets are
    rounded to `dtype` first, and the codes chosen for them as rounded."""
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError(f"quantize_int4 takes a 2-D floating-point weight, got {tuple(weight.shape)} {weight.dtype}")
    if group_size not in GROUP_SIZES or weight.shape[1] % group_size or weight.numel() == 0:
        raise ValueError(f"group size {group_size} of {GROUP_SIZES} must divide the {weight.shape[1]} columns")
    if dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"scales are bfloat16 or float32, not {dtype}")
    rows, cols = weight.shape
    v = weight.detach().float().view(rows, cols // group_size, group_size)
    if not bool(torch.isfinite(v).all()):
        raise ValueError("the weight holds infinities or NaN")
    low, high = v.amin(2), v.amax(2)
    scales = (torch.maximum(high / 7, -low / 8) if symmetric else (high - low) / 15).to(dtype)
    scales = torch.where(scales == 0, torch.ones_like(scales), scales)
    offsets = None if symmetric else low.to(dtype)
    base = -8 * scales.float() if symmetric else offsets.float()
    if not bool(torch.isfinite(base).all()) or not bool(torch.isfinite(base + 15 * scales.float()).all()):
        raise ValueError(f"the weight's range does not fit {dtype} scales and offsets")
    q = ((v - base[:, :, None]) / scales.float()[:, :, None]).round_().clamp_(0, 15).to(torch.uint8).view(rows, cols)
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), scales, offsets


class Int4Linear(torch.nn.Module):
    """``nn.Linear`` ABI over 4-bit codes, scales and offsets."""

    def __init__(self, in_features: int, out_features: int, *, group_size: int = 64, symmetric: bool = False,
                 bias: bool = False, device=None, dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        if group_size not in GROUP_SIZES or in_features % group_size:
            raise ValueError(f"group size {group_size} of {GROUP_SIZES} must divide in_features {in_features}")
        self.in_features, self.out_features, self.group_size = int(in_features), int(out_features), int(group_size)
        tables = (out_features, in_features // group_size)
        self.register_buffer("weight", torch.zeros((out_features, in_features // 2), dtype=torch.uint8, device=device))
        self.register_buffer("scales", torch.ones(tables, dtype=dtype, device=device))
        self.register_buffer("offsets", None if symmetric else torch.zeros(tables, dtype=dtype, device=device))
        self.register_buffer("bias", torch.zeros(out_features, dtype=dtype, device=device) if bias else None)

    @classmethod
    def from_weight(cls, weight: torch.Tensor, bias: torch.Tensor | None = None, *, group_size: int = 64,
                    symmetric: bool = False, dtype: torch.dtype = torch.bfloat16) -> "Int4Linear":
        codes, scales, offsets = quantize_int4(weight, group_size, symmetric, dtype)
        layer = cls(weight.shape[1], weight.shape[0], group_size=group_size, symmetric=symmetric, device="meta",
                    dtype=dtype)
        layer.weight, layer.scales, layer.offsets = codes, scales, offsets
        layer.bias = None if bias is None else bias.detach().to(dtype)
        return layer

    @classmethod
    def from_linear(cls, linear, **options) -> "Int4Linear":
        return cls.from_weight(linear.weight, getattr(linear, "bias", None), **options)

    def forward(self, x):
        return int4_linear(x, self.weight, self.scales, self.offsets, self.bias)


def native_joined_swiglu(joined: torch.Tensor, limit: float) -> torch.Tensor:
    """The native call behind glm53::joined_swiglu: the clamped SwiGLU of
    bfloat16 [..., 2 I] rows, gate first."""
    joined = joined.contiguous()
    width = joined.shape[-1] // 2
    h = torch.empty((*joined.shape[:-1], width), dtype=torch.bfloat16, device=joined.device)
    N.run(joined.get_device(), N.lib().glm53_activate_gate_up, joined.data_ptr(), h.numel() // width, width, limit, h.data_ptr())
    return h


class Int4MLP(torch.nn.Module):
    """Gated MLP over 4-bit weights: one product for gate and up (stacked, gate
    rows first), the package's clamped SwiGLU with its bf16 rounding steps,
    and the down projection."""

    def __init__(self, gate_up_proj: Int4Linear, down_proj: Int4Linear, limit: float | None = None):
        super().__init__()
        if gate_up_proj.out_features != 2 * down_proj.in_features:
            raise ValueError(f"gate and up rows {gate_up_proj.out_features} != 2 x {down_proj.in_features}")
        self.gate_up_proj, self.down_proj = gate_up_proj, down_proj
        self.limit = limit

    @classmethod
    def from_weights(cls, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, limit: float | None = None,
                     **options) -> "Int4MLP":
        if gate.shape != up.shape or down.shape != gate.t().shape:
            raise ValueError(f"shapes do not match: gate {tuple(gate.shape)}, up {tuple(up.shape)}, "
                             f"down {tuple(down.shape)}")
        return cls(Int4Linear.from_weight(torch.cat([gate.detach(), up.detach()]), **options),
                   Int4Linear.from_weight(down, **options), limit)

    def forward(self, x):
        limit = math.inf if self.limit is None else float(self.limit)
        if not limit > 0:
            raise ValueError(f"limit must be positive, got {limit}")
        joined = self.gate_up_proj(x)
        if _ops.direct(joined):
            return self.down_proj(native_joined_swiglu(joined, limit))
        _ops.refuse_transforms("Int4MLP", joined)
        return self.down_proj(torch.ops.glm53.joined_swiglu(joined, limit))
