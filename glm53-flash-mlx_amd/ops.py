"""The path's entry points as torch.library custom ops.

The native library is called through ctypes, which torch.compile cannot
trace: every MoE call would break the graph.  Registered as custom ops
(namespace ``glm53``) with shape functions, each call is one opaque node --
``torch.compile(..., fullgraph=True)`` traces a model through the MoE layers,
and FakeTensor / meta propagation gets the output shapes without a device.

* ``glm53::block_fp8_linear(x, weight, scale_inv, code_flags?)`` -- fp8.py
  ``block_fp8_linear``;
* ``glm53::router_topk(x, weight, bias, top_k, routed_scaling_factor,
  norm_topk_prob, n_group, topk_group)`` -- ``Float32Gate``;
* ``glm53::moe_decode(x, owner, expert_ids?, scores?)`` -- one token through
  a ``PackedFP8MoE`` (router + routed + shared, or caller routing);
* ``glm53::moe_prefill(x, owner, expert_ids?, scores?)`` -- the grouped
  prefill of a ``SortedGroupedFP8MoE``;
* ``glm53::moe_direct(x, owner)`` -- a batch below a ``SortedGroupedFP8MoE``'s
  min_routes as one prefill in the Direct order;
* ``glm53::residual_norm(residual, out?, post_weight?, gate?, next_weight?,
  ...)`` and ``glm53::residual_norm_backward`` -- ``rms_norm`` (without out)
  and ``residual_norm``, differentiable;
* ``glm53::gated_mlp(x, gate_weight, up_weight, down_weight, limit, keep)``
  and ``glm53::gated_mlp_backward`` -- ``gated_mlp``, differentiable where
  `keep` has it return G, U and h;
* ``glm53::int4_linear(x, weight, scales, offsets?, bias?)`` -- ``int4_linear``,
  and ``glm53::joined_swiglu(joined, limit)``, the activation of ``Int4MLP``.

The MoE ops take the module by an integer key (``register_owner``): the
module keeps its weights, its per-(device, stream) native plans and its
cached 0x7F/0xFF code flags, as an ``nn.Module`` does for its parameters,
and the op reads them from there.  Outputs are always new tensors.
"""

from __future__ import annotations

import itertools
import weakref
from typing import Optional

import torch

_OWNERS: dict[int, weakref.ref] = {}
_KEYS = itertools.count(1)


def register_owner(module) -> int:
    """A key under which the MoE ops find `module` (held weakly)."""
    key = next(_KEYS)
    _OWNERS[key] = weakref.ref(module)
    return key


_PLAIN_TENSORS = (torch.Tensor, torch.nn.Parameter, torch.nn.Buffer)


def _dispatch_probe():
    """A function that tells whether anything acts between an eager call and
    its kernel.  It asks torch's private state; where this torch lacks one of
    the names, the function says yes and every call goes through the op."""
    try:
        c, forward_ad, profiling = torch._C, torch.autograd.forward_ad, torch.autograd._profiler_enabled
        tracing, transforms = c._get_tracing_state, c._functorch.peek_interpreter_stack
        dispatch_modes, function_modes = c._len_torch_dispatch_stack, c._len_torch_function_stack
        forward_ad._current_level
    except AttributeError:
        return lambda: True

    def acts() -> bool:
        return bool(torch.compiler.is_compiling() or tracing() is not None or dispatch_modes() or function_modes()
                    or transforms() is not None or forward_ad._current_level >= 0 or profiling())

    return acts


_dispatch_acts = _dispatch_probe()


def direct(*tensors) -> bool:
    """True when dispatching an op on `tensors` could only reach its device
    kernel, so that an eager call may run the native call itself: the custom
    op's Python layers cost ~12 us a call, more than a one-row linear's
    kernel (4.5 us) and its launch together (call of a 4096 x 4096
    BlockFP8Linear: 20 us through the op, 11 us direct).  Anything that
    acts between the call and the kernel goes through the op: tracing and
    compilation, dispatch and function modes, functorch transforms, forward-
    and reverse-mode differentiation, a recording profiler, tensor
    subclasses."""
    if _dispatch_acts():
        return False
    grad = torch.is_grad_enabled()
    for t in tensors:
        if t is not None and (type(t) not in _PLAIN_TENSORS or (grad and t.requires_grad)):
            return False
    return True


def eager(*tensors) -> bool:
    """As ``direct``, but with reverse-mode differentiation allowed: a call
    that nothing else acts on may run as a torch.autograd.Function."""
    return not _dispatch_acts() and all(t is None or type(t) in _PLAIN_TENSORS for t in tensors)


def _carries_derivative(t: torch.Tensor) -> bool:
    """Whether `t` carries a tangent or a gradient of torch.func at any of the
    levels that are active: asked level by level from the innermost one, below
    which its wrapper is taken off and the level left."""
    functorch, forward_ad = torch._C._functorch, torch.autograd.forward_ad
    top = functorch.peek_interpreter_stack()
    if top is None or torch.compiler.is_compiling():
        return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None
    if functorch.is_functorch_wrapped_tensor(t) and functorch.maybe_get_level(t) == top.level():
        if functorch.is_gradtrackingtensor(t):
            if top.key() == functorch.TransformType.Jvp:
                carries = forward_ad.unpack_dual(t).tangent is not None
            else:
                carries = t.requires_grad
            if carries:
                return True
        t = functorch.get_unwrapped(t)
    from torch._functorch import pyfunctorch

    with pyfunctorch.temporarily_pop_interpreter_stack():
        return _carries_derivative(t)


def refuse_transforms(what: str, *tensors) -> None:
    """An error where one of `tensors` carries a derivative that a custom op
    would drop or cannot give: a forward-mode tangent (dropped below autograd,
    the result's tangent would be zero), or torch.func's own differentiation.
    Before a call that ``direct`` and ``eager`` leave to the op."""
    if torch.autograd.forward_ad._current_level < 0 and (torch.compiler.is_compiling()
                                                         or torch._C._functorch.peek_interpreter_stack() is None):
        return
    for t in tensors:
        if t is not None and _carries_derivative(t):
            raise RuntimeError(f"{what} has no derivative in forward mode or under torch.func: "
                               "use torch.autograd in reverse mode")


def _owner(key: int):
    ref = _OWNERS.get(int(key))
    module = ref() if ref is not None else None
    if module is None:
        raise RuntimeError(f"MoE module {key} no longer exists")
    return module


@torch.library.custom_op("glm53::block_fp8_linear", mutates_args=())
def block_fp8_linear(x: torch.Tensor, weight: torch.Tensor, scale_inv: torch.Tensor,
                     code_flags: Optional[torch.Tensor]) -> torch.Tensor:
    from .fp8 import native_block_fp8_linear

    return native_block_fp8_linear(x, weight, scale_inv, code_flags)


@block_fp8_linear.register_fake
def _(x, weight, scale_inv, code_flags):
    return x.new_empty((*x.shape[:-1], weight.shape[0]))


@torch.library.custom_op("glm53::router_topk", mutates_args=())
def router_topk(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, top_k: int, routed_scaling_factor: float,
                norm_topk_prob: bool, n_group: int = 1, topk_group: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    from .router import native_router_topk

    return native_router_topk(x, weight, bias, top_k, routed_scaling_factor, norm_topk_prob, n_group, topk_group)


@router_topk.register_fake
def _(x, weight, bias, top_k, routed_scaling_factor, norm_topk_prob, n_group=1, topk_group=1):
    lead = x.shape[:-1]
    return (x.new_empty((*lead, top_k), dtype=torch.int32), x.new_empty((*lead, top_k), dtype=torch.float32))


@torch.library.custom_op("glm53::moe_decode", mutates_args=())
def moe_decode(x: torch.Tensor, owner: int, expert_ids: Optional[torch.Tensor],
               scores: Optional[torch.Tensor]) -> torch.Tensor:
    return _owner(owner).native_decode(x, expert_ids, scores)


@moe_decode.register_fake
def _(x, owner, expert_ids, scores):
    return torch.empty_like(x)


@torch.library.custom_op("glm53::moe_prefill", mutates_args=())
def moe_prefill(x: torch.Tensor, owner: int, expert_ids: Optional[torch.Tensor],
                scores: Optional[torch.Tensor]) -> torch.Tensor:
    return _owner(owner).native_prefill(x, expert_ids, scores)


@moe_prefill.register_fake
def _(x, owner, expert_ids, scores):
    return torch.empty_like(x)


@torch.library.custom_op("glm53::moe_direct", mutates_args=())
def moe_direct(x: torch.Tensor, owner: int) -> torch.Tensor:
    return _owner(owner).native_direct(x)


@moe_direct.register_fake
def _(x, owner):
    return torch.empty_like(x)


@torch.library.custom_op("glm53::residual_norm", mutates_args=())
def residual_norm(residual: torch.Tensor, out: Optional[torch.Tensor], post_weight: Optional[torch.Tensor],
                  gate: Optional[torch.Tensor], next_weight: Optional[torch.Tensor], kind: int, rows_per_gate: int,
                  scale: float, eps: float, normed: bool,
                  y_f32: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    from .norms import native_residual_norm

    x, y, stats = native_residual_norm(residual, out, post_weight, gate, next_weight, kind, rows_per_gate, scale, eps,
                                       normed, y_f32)
    y_type = torch.float32 if y_f32 else torch.bfloat16
    return (residual.new_empty(0) if x is None else x, residual.new_empty(0, dtype=y_type) if y is None else y, stats)


@residual_norm.register_fake
def _(residual, out, post_weight, gate, next_weight, kind, rows_per_gate, scale, eps, normed, y_f32):
    y_type = torch.float32 if y_f32 else torch.bfloat16
    rows = residual.numel() // residual.shape[-1]
    return (residual.new_empty(residual.shape if out is not None else 0),
            residual.new_empty(residual.shape if normed else 0, dtype=y_type),
            residual.new_empty((rows, 2), dtype=torch.float32))


@torch.library.custom_op("glm53::residual_norm_backward", mutates_args=())
def residual_norm_backward(residual: torch.Tensor, out: Optional[torch.Tensor], post_weight: Optional[torch.Tensor],
                           gate: Optional[torch.Tensor], next_weight: Optional[torch.Tensor], stats: torch.Tensor,
                           d_new: Optional[torch.Tensor], d_y: Optional[torch.Tensor], kind: int, rows_per_gate: int,
                           scale: float, eps: float, y_f32: bool, wanted: list[bool]) -> list[torch.Tensor]:
    from .norms import native_residual_norm_backward

    grads = native_residual_norm_backward(residual, out, post_weight, gate, next_weight, stats, d_new, d_y, kind,
                                          rows_per_gate, scale, eps, y_f32, wanted)
    return [residual.new_empty(0) if g is None else g for g in grads]


@residual_norm_backward.register_fake
def _(residual, out, post_weight, gate, next_weight, stats, d_new, d_y, kind, rows_per_gate, scale, eps, y_f32, wanted):
    inputs = (residual, out, post_weight, gate, next_weight)
    return [t.new_empty(t.shape) if t is not None and w else residual.new_empty(0) for t, w in zip(inputs, wanted)]


def _residual_norm_context(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:5], output[2])
    ctx.form = inputs[5:]
    ctx.set_materialize_grads(False)


def _residual_norm_backward(ctx, d_new, d_y, _):
    saved = ctx.saved_tensors
    kind, rows_per_gate, scale, eps, normed, y_f32 = ctx.form
    wanted = [bool(w) for w in ctx.needs_input_grad[:5]]
    grads = torch.ops.glm53.residual_norm_backward(*saved, d_new if saved[1] is not None else None,
                                                   d_y if normed else None, kind, rows_per_gate, scale, eps, y_f32,
                                                   wanted)
    return (*(g if w else None for g, w in zip(grads, wanted)), None, None, None, None, None, None)


residual_norm.register_autograd(_residual_norm_backward, setup_context=_residual_norm_context)


@torch.library.custom_op("glm53::gated_mlp", mutates_args=())
def gated_mlp(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor, down_weight: torch.Tensor,
              limit: float, keep: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    from .gated import native_gated_mlp

    y, gate, up, h = native_gated_mlp(x, gate_weight, up_weight, down_weight, limit, keep)
    if keep:
        return y, gate, up, h
    return y, x.new_empty(0, dtype=torch.float32), x.new_empty(0, dtype=torch.float32), x.new_empty(0)


@gated_mlp.register_fake
def _(x, gate_weight, up_weight, down_weight, limit, keep):
    from .gated import FEW_ROWS

    rows = x.numel() // x.shape[-1]
    kept = (rows, gate_weight.shape[0]) if keep else (0,)
    return (x.new_empty(x.shape), x.new_empty(kept, dtype=torch.float32), x.new_empty(kept, dtype=torch.float32),
            x.new_empty((2, *kept) if keep and rows <= FEW_ROWS else kept))


@torch.library.custom_op("glm53::gated_mlp_backward", mutates_args=())
def gated_mlp_backward(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor, down_weight: torch.Tensor,
                       gate: torch.Tensor, up: torch.Tensor, h: torch.Tensor, d_y: torch.Tensor, limit: float,
                       wanted: list[bool]) -> list[torch.Tensor]:
    from .gated import native_gated_mlp_backward

    grads = native_gated_mlp_backward(x, gate_weight, up_weight, down_weight, gate, up, h, d_y, limit, wanted)
    return [x.new_empty(0) if g is None else g for g in grads]


@gated_mlp_backward.register_fake
def _(x, gate_weight, up_weight, down_weight, gate, up, h, d_y, limit, wanted):
    inputs = (x, gate_weight, up_weight, down_weight)
    return [t.new_empty(t.shape) if w else x.new_empty(0) for t, w in zip(inputs, wanted)]


def _gated_mlp_context(ctx, inputs, output):
    if not inputs[5]:
        raise RuntimeError("glm53::gated_mlp without keep has no gradient")
    ctx.save_for_backward(*inputs[:4], *output[1:])
    ctx.limit = inputs[4]
    ctx.set_materialize_grads(False)


def _gated_mlp_backward(ctx, d_y, _gate, _up, _h):
    if d_y is None:
        return (None,) * 6
    wanted = [bool(w) for w in ctx.needs_input_grad[:4]]
    grads = torch.ops.glm53.gated_mlp_backward(*ctx.saved_tensors, d_y, ctx.limit, wanted)
    return (*(g if w else None for g, w in zip(grads, wanted)), None, None)


gated_mlp.register_autograd(_gated_mlp_backward, setup_context=_gated_mlp_context)


@torch.library.custom_op("glm53::int4_linear", mutates_args=())
def int4_linear(x: torch.Tensor, weight: torch.Tensor, scales: torch.Tensor, offsets: Optional[torch.Tensor],
                bias: Optional[torch.Tensor]) -> torch.Tensor:
    from .int4 import native_int4_linear

    return native_int4_linear(x, weight, scales, offsets, bias)


@int4_linear.register_fake
def _(x, weight, scales, offsets, bias):
    return x.new_empty((*x.shape[:-1], weight.shape[0]))


@torch.library.custom_op("glm53::joined_swiglu", mutates_args=())
def joined_swiglu(joined: torch.Tensor, limit: float) -> torch.Tensor:
    from .int4 import native_joined_swiglu

    return native_joined_swiglu(joined, limit)


@joined_swiglu.register_fake
def _(joined, limit):
    return joined.new_empty((*joined.shape[:-1], joined.shape[-1] // 2))
