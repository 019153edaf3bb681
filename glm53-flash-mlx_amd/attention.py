"""Attention within packed sequences, with gradients.

    S = scale q k^T over the keys a query sees, P = softmax(S), out = P v

Sequences of different lengths lie one behind the other in one tensor; query
head h reads key head h / (heads / kv_heads).  Scores, the softmax and all sums
are FP32; P, and in the gradients dS, are rounded to bf16 once as operands of
the products that take them, and each result once.  A call that may be
differentiated keeps 4 bytes a row for its gradients, whatever the lengths.
The reference's attention is sparse and recurrent and has no counterpart.
"""

from __future__ import annotations

import ctypes

import torch

from . import _native as N
from . import ops as _ops

MAX_HEAD_DIM = 256
MAX_STRIDE = 1 << 22  # elements from one token, or one head, to the next
MAX_HEAD_SPAN = 1 << 30  # of a token's heads together
MIN_SCALE, MAX_SCALE = 2.0**-64, 2.0**127  # the largest: its product with log2 e is an FP32 number


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor | None = None,
                     key_offsets: torch.Tensor | None = None, *, causal: bool = True,
                     scale: float | None = None) -> torch.Tensor:
    """Attention of q bfloat16 [tokens, heads, dim] over k and v bfloat16
    [keys, kv_heads, dim]; the result has q's shape.

    offsets int32 [sequences + 1], ascending, on the device: sequence s is
    tokens offsets[s] .. offsets[s + 1] - 1 (None: all are one sequence).
    key_offsets: the same for keys, where they are not the queries' own (a
    chunk of a prompt over all of its keys).  causal: the last query of a sequence
    sees all of its keys, each one before it one key less.  Queries that see no key,
    and rows of no sequence, are 0, those whose largest scaled score is beyond FP32 NaN.
    scale: 1 / sqrt(dim) where None, 2^-64 to 2^127.

    heads a multiple of kv_heads, dim a multiple of 8 up to 256.  q, k and v
    may be views of one tensor (a joint projection's) without a copy.
    Differentiable in q, k and v (first order, in reverse mode; forward mode and
    torch.func's grad, vjp and jvp raise)."""
    N.same_device(q, k, v, offsets, key_offsets)
    check_heads(q, k, v)
    dim = q.shape[2]
    for name, t in (("offsets", offsets), ("key_offsets", key_offsets)):
        check_offsets(name, t)
    if key_offsets is not None and (offsets is None or offsets.shape != key_offsets.shape):
        raise ValueError("key_offsets need offsets of the same number of sequences")
    if key_offsets is None and q.shape[0] != k.shape[0]:
        raise ValueError(f"{k.shape[0]} keys for {q.shape[0]} queries need key_offsets")
    scale = check_scale(scale, dim)
    if _ops.direct(q, k, v):
        return native_packed_attention(q, k, v, offsets, key_offsets, bool(causal), scale, False)[0]
    if _ops.eager(q, k, v):
        return _PackedAttention.apply(q, k, v, offsets, key_offsets, bool(causal), scale)
    _ops.refuse_transforms("packed_attention", q, k, v)
    keep = torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v))
    return torch.ops.glm53.packed_attention(q, k, v, offsets, key_offsets, bool(causal), scale, keep)[0]


def check_heads(q: torch.Tensor, *others: torch.Tensor) -> None:
    """q [n, heads, dim] and keys or values [m, kv_heads, dim], bfloat16."""
    for t in (q, *others):
        if t.dtype is not torch.bfloat16 or t.dim() != 3:
            raise ValueError(f"attention takes bfloat16 [rows, heads, dim] tensors, got {tuple(t.shape)} {t.dtype}")
    heads, dim = q.shape[1:]
    for t in others:
        if t.shape != others[0].shape or t.shape[2] != dim or t.shape[1] == 0 or heads == 0 or heads % t.shape[1]:
            raise ValueError(f"shapes do not match: q {tuple(q.shape)}, k and v {[tuple(o.shape) for o in others]}")
    check_dim(dim)


def check_dim(dim: int) -> None:
    if dim == 0 or dim % 8 or dim > MAX_HEAD_DIM:
        raise ValueError(f"head dim {dim} must be a multiple of 8 up to {MAX_HEAD_DIM}")


def check_offsets(name: str, t: torch.Tensor | None) -> None:
    if t is not None and (t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] < 2):
        raise ValueError(f"{name} must be int32 [sequences + 1], got {tuple(t.shape)} {t.dtype}")


def check_scale(scale: float | None, dim: int) -> float:
    scale = dim**-0.5 if scale is None else float(scale)
    if not MIN_SCALE <= scale <= MAX_SCALE:
        raise ValueError(f"scale must be from 2^-64 to 2^127, got {scale}")
    return scale


def head_rows(t: torch.Tensor) -> tuple[torch.Tensor, N.HeadRows]:
    """A [rows, heads, dim] tensor as the kernels take it, and their view of
    it: any strides that are multiples of 8 elements, or a copy."""
    rows, heads, dim = t.shape
    row, head, one = t.stride()
    if rows == 1:
        row = 0
    if heads == 1:
        head = 0
    if one != 1 or (row | head) & 7 or max(row, head) > MAX_STRIDE or heads * head > MAX_HEAD_SPAN or t.data_ptr() & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        row, head = heads * dim, dim
    return t, N.HeadRows(t.data_ptr(), row, head)


def result_like(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape; for a contiguous one by the call that is 0.6 us shorter."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def index_pointer(t: torch.Tensor | None) -> tuple[torch.Tensor | None, int | None]:
    if t is None:
        return None, None
    t = t.contiguous()
    return t, t.data_ptr()


def _descriptor(q, k, v, offsets, key_offsets, out, lse, causal, scale):
    """The call's descriptor, and what has to live until it is made."""
    (q, q_rows), (k, k_rows), (v, v_rows) = map(head_rows, (q, k, v))
    offsets, p_offsets = index_pointer(offsets)
    key_offsets, p_key_offsets = index_pointer(key_offsets)
    d = N.Attention(q.shape[0], k.shape[0], 0 if offsets is None else offsets.shape[0] - 1, q.shape[1], k.shape[1],
                    q.shape[2], q_rows, k_rows, v_rows, p_offsets, p_key_offsets, out.data_ptr(),
                    None if lse is None else lse.data_ptr())
    d.causal, d.scale = causal, scale
    return d, (q, k, v, offsets, key_offsets)


def native_packed_attention(q, k, v, offsets, key_offsets, causal: bool, scale: float, keep: bool):
    """The native call behind glm53::packed_attention: the result, and the
    rows' logarithms where kept."""
    tokens, heads, _ = q.shape
    out = result_like(q)
    lse = q.new_empty((k.shape[1], tokens * (heads // k.shape[1])), dtype=torch.float32) if keep else None
    if tokens:
        d, alive = _descriptor(q, k, v, offsets, key_offsets, out, lse, causal, scale)
        N.run(q.get_device(), N.lib().glm53_packed_attention, ctypes.byref(d))
    return out, lse


def native_packed_attention_backward(q, k, v, offsets, key_offsets, out, lse, d_out, causal: bool, scale: float,
                                     wanted: list[bool]):
    """The native call behind glm53::packed_attention_backward: the gradients
    of q, k and v that are `wanted`, None in place of the others."""
    grads = [result_like(t) if w else None for t, w in zip((q, k, v), wanted)]
    if q.shape[0] == 0 or k.shape[0] == 0:
        return [None if g is None else g.zero_() for g in grads]
    d, alive = _descriptor(q, k, v, offsets, key_offsets, out, lse, causal, scale)
    d_out, d.d_out = head_rows(d_out)
    d.d_q, d.d_k, d.d_v = (None if g is None else g.data_ptr() for g in grads)
    lib = N.lib()
    d.workspace_bytes = lib.glm53_packed_attention_backward_workspace_bytes(q.shape[0], q.shape[1])
    if wanted[1] or wanted[2]:
        d.workspace_bytes += lib.glm53_packed_attention_backward_split_bytes(d.tokens, d.keys, d.sequences, d.heads, d.kv_heads,
                                                                             d.head_dim)
    ws = N.workspace(d.workspace_bytes, q.device)
    d.workspace = ws.data_ptr()
    N.run(q.get_device(), lib.glm53_packed_attention_backward, ctypes.byref(d))
    return grads


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, key_offsets, causal, scale):
        out, lse = native_packed_attention(q, k, v, offsets, key_offsets, causal, scale, True)
        ctx.save_for_backward(q, k, v, offsets, key_offsets, out, lse)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        return (*native_packed_attention_backward(*ctx.saved_tensors, d_out, ctx.causal, ctx.scale,
                                                  ctx.needs_input_grad[:3]), None, None, None, None)
