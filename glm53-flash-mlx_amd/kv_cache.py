"""A paged key-value cache, and one token's attention over it.

A cache is pages of `page_size` tokens, [pages, kv_heads, page_size, dim] for
keys and the same for values, and a sequence is the pages that its row of a
page table names: token `position` lies in page_table[s, position /
page_size].  Rows are bfloat16, or E4M3 codes (uint8) with one power of two a row,
[pages, kv_heads, page_size] bytes 127 + e:

    value = code * 2^e,  e the smallest with |x| <= 448 * 2^e for the row's x

E4M3 has an exponent of its own, so a row's power of two only has to bring it
into range; it costs no precision that a finer scale would keep, and every
value that a cache holds is a bfloat16 value (the largest bfloat16 numbers, which
a code would round to 2^128, are stored as 240 * 2^120): reading back is exact.  An
infinity or NaN is stored as NaN.  Half the bytes of a bfloat16 cache, and a
token's attention over a cache takes the time of its bytes.

Nothing here has gradients, and nothing is read back to the host: lengths and
tables stay on the device, so a step can be captured once and replayed
while they change.
"""

from __future__ import annotations

import ctypes

import torch

from . import _native as N
from . import ops as _ops
from .attention import check_dim, check_heads, check_offsets, check_scale, head_rows, index_pointer, result_like


def append_kv(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
              lengths: torch.Tensor, offsets: torch.Tensor | None = None, *, k_scales: torch.Tensor | None = None,
              v_scales: torch.Tensor | None = None) -> None:
    """Writes new tokens' keys and values into the pages of their sequences.

    k, v bfloat16 [tokens, kv_heads, dim]; page_table int32 [sequences, pages
    of a sequence]; lengths int32 [sequences]: what each holds already; offsets
    int32 [sequences + 1]: sequence s's new tokens, None: one each.  A token
    whose place has no page, or one outside the cache, is left out; so are rows
    of no sequence.  Pages that several sequences share are not to be written to."""
    N.same_device(k, v, k_pages, v_pages, page_table, lengths, offsets, k_scales, v_scales)
    _check_cache(k_pages, v_pages, page_table, k_scales, v_scales)
    check_heads(k, v)
    if k.shape != v.shape or k.shape[1:] != (k_pages.shape[1], k_pages.shape[3]):
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not fit pages {tuple(k_pages.shape)}")
    _check_lengths("lengths", lengths, page_table)
    _check_sequences(offsets, page_table)
    if offsets is None and k.shape[0] != page_table.shape[0]:
        raise ValueError(f"{k.shape[0]} tokens for {page_table.shape[0]} sequences need offsets")
    tensors = (k.detach(), v.detach(), k_pages, v_pages, page_table, lengths, offsets, k_scales, v_scales)
    if _ops.direct(*tensors):
        native_append_kv(*tensors)
        return
    _ops.refuse_transforms("append_kv", k, v)
    torch.ops.glm53.append_kv(*tensors)


def read_kv(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, offsets: torch.Tensor, rows: int, *,
            k_scales: torch.Tensor | None = None,
            v_scales: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of whole sequences, packed: bfloat16 [rows, kv_heads,
    dim] each, sequence s's first offsets[s + 1] - offsets[s] tokens from row
    offsets[s] on, as ``packed_attention`` takes them.  Rows of no sequence
    are 0, tokens without a page in the cache NaN."""
    N.same_device(k_pages, v_pages, page_table, offsets, k_scales, v_scales)
    _check_cache(k_pages, v_pages, page_table, k_scales, v_scales)
    if offsets is None:
        raise ValueError("read_kv needs offsets")
    _check_sequences(offsets, page_table)
    if rows < 0:
        raise ValueError(f"rows must not be negative, got {rows}")
    tensors = (k_pages, v_pages, page_table, offsets, int(rows), k_scales, v_scales)
    if _ops.direct(k_pages, v_pages):
        return native_read_kv(*tensors)
    _ops.refuse_transforms("read_kv", k_pages, v_pages)
    return torch.ops.glm53.read_kv(*tensors)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, *, k_scales: torch.Tensor | None = None, v_scales: torch.Tensor | None = None,
                    scale: float | None = None) -> torch.Tensor:
    """Attention of one token a sequence, q bfloat16 [sequences, heads, dim],
    over that sequence's first lengths[s] tokens in the cache.

    lengths int32 [sequences].  A sequence without a token gives 0, one with a
    token that has no page in the cache NaN, and so does a head whose largest scaled
    score is beyond FP32.  scale: 1 / sqrt(dim) where None, 2^-64 to 2^127.
    The softmax and all sums are FP32, its weights are rounded to bf16 as
    operands, the result once."""
    N.same_device(q, k_pages, v_pages, page_table, lengths, k_scales, v_scales)
    _check_cache(k_pages, v_pages, page_table, k_scales, v_scales)
    check_heads(q)
    kv_heads, dim = k_pages.shape[1], k_pages.shape[3]
    if q.shape[2] != dim or q.shape[1] == 0 or q.shape[1] % kv_heads or q.shape[0] != page_table.shape[0]:
        raise ValueError(f"q {tuple(q.shape)} does not fit {page_table.shape[0]} sequences of pages {tuple(k_pages.shape)}")
    _check_lengths("lengths", lengths, page_table)
    tensors = (q, k_pages, v_pages, page_table, lengths, k_scales, v_scales, check_scale(scale, dim))
    if _ops.direct(q, k_pages, v_pages):
        return native_paged_attention(*tensors)
    _ops.refuse_transforms("paged_attention", q, k_pages, v_pages)
    return torch.ops.glm53.paged_attention(*tensors)


def _check_cache(k_pages, v_pages, page_table, k_scales, v_scales) -> None:
    shape, kind = k_pages.shape, k_pages.dtype
    if kind not in (torch.bfloat16, torch.uint8) or v_pages.dtype is not kind or len(shape) != 4 or v_pages.shape != shape:
        raise ValueError("a cache's pages are two bfloat16 or uint8 [pages, kv_heads, page_size, dim] tensors, got "
                         f"{tuple(shape)} {kind} and {tuple(v_pages.shape)} {v_pages.dtype}")
    if not k_pages.is_contiguous() or not v_pages.is_contiguous() or (k_pages.data_ptr() | v_pages.data_ptr()) & 15:
        raise ValueError("a cache's pages must be contiguous and 16-byte aligned")
    pages, kv_heads, page_size, dim = shape
    if pages == 0 or kv_heads == 0:
        raise ValueError(f"a cache needs pages and heads, got {tuple(shape)}")
    if page_size < 16 or page_size > 65536 or page_size & (page_size - 1):
        raise ValueError(f"page size {page_size} must be a power of two from 16 to 65536")
    check_dim(dim)
    quantised = kind is torch.uint8
    if quantised and dim % 16:
        raise ValueError(f"an E4M3 cache needs a head dim that is a multiple of 16, got {dim}")
    for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
        if (t is not None) != quantised:
            raise ValueError(f"{name} belong to an E4M3 cache")
        if t is not None and (t.dtype is not torch.uint8 or t.shape != shape[:3] or not t.is_contiguous() or t.data_ptr() & 15):
            raise ValueError(f"{name} must be a contiguous, 16-byte aligned uint8 {tuple(shape[:3])} tensor")
    if page_table.dtype is not torch.int32 or page_table.dim() != 2:
        raise ValueError(f"page_table must be int32 [sequences, pages], got {tuple(page_table.shape)} {page_table.dtype}")


def _check_lengths(name, lengths, page_table) -> None:
    if lengths.dtype is not torch.int32 or lengths.shape != page_table.shape[:1]:
        raise ValueError(f"{name} must be int32 [{page_table.shape[0]}], got {tuple(lengths.shape)} {lengths.dtype}")


def _check_sequences(offsets, page_table) -> None:
    if offsets is None:
        return
    check_offsets("offsets", offsets)
    if offsets.shape[0] != page_table.shape[0] + 1:
        raise ValueError(f"{offsets.shape[0]} offsets for {page_table.shape[0]} sequences")


def _descriptor(k_pages, v_pages, page_table, k_scales, v_scales):
    """The cache's descriptor, and the table that has to live until the call is made."""
    if page_table.shape[1] and page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    pages, kv_heads, page_size, dim = k_pages.shape
    sequences, most = page_table.shape
    quantised = k_scales is not None
    return N.KVCache(k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr() if quantised else None,
                     v_scales.data_ptr() if quantised else None, page_table.data_ptr(), pages, page_size, kv_heads, dim,
                     sequences, most, page_table.stride(0) if sequences > 1 else most, quantised), page_table


def native_append_kv(k, v, k_pages, v_pages, page_table, lengths, offsets, k_scales, v_scales) -> None:
    """The native call behind glm53::append_kv."""
    cache, table = _descriptor(k_pages, v_pages, page_table, k_scales, v_scales)
    (k, k_rows), (v, v_rows) = head_rows(k), head_rows(v)
    offsets, p_offsets = index_pointer(offsets)
    lengths, p_lengths = index_pointer(lengths)
    if k.shape[0] and table.shape[0]:
        N.run(k.get_device(), N.lib().glm53_kv_append, ctypes.byref(cache), ctypes.byref(k_rows), ctypes.byref(v_rows),
              k.shape[0], p_offsets, p_lengths)


def native_read_kv(k_pages, v_pages, page_table, offsets, rows: int, k_scales, v_scales):
    """The native call behind glm53::read_kv."""
    cache, table = _descriptor(k_pages, v_pages, page_table, k_scales, v_scales)
    shape = (rows, k_pages.shape[1], k_pages.shape[3])
    k, v = (k_pages.new_empty(shape, dtype=torch.bfloat16) for _ in range(2))
    offsets, p_offsets = index_pointer(offsets)
    if rows:
        N.run(k.get_device(), N.lib().glm53_kv_read, ctypes.byref(cache), p_offsets, rows, k.data_ptr(), v.data_ptr())
    return k, v


def native_paged_attention(q, k_pages, v_pages, page_table, lengths, k_scales, v_scales, scale: float):
    """The native call behind glm53::paged_attention."""
    cache, table = _descriptor(k_pages, v_pages, page_table, k_scales, v_scales)
    out = result_like(q)
    q, q_rows = head_rows(q)
    lengths, p_lengths = index_pointer(lengths)
    sequences, heads, dim = q.shape
    if sequences:
        lib = N.lib()
        ws_bytes = lib.glm53_paged_attention_workspace_bytes(dim, k_scales is not None)
        ws = N.workspace(ws_bytes, q.device)
        N.run(q.get_device(), lib.glm53_paged_attention, ctypes.byref(cache), ctypes.byref(q_rows), heads, p_lengths, scale,
              out.data_ptr(), ws.data_ptr(), ws_bytes)
    return out
