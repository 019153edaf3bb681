"""Self-attention as a module beside the feed-forwards: projections around
``packed_attention`` in training and over a prompt, around the key-value
cache in serving.  No positions are encoded."""

from __future__ import annotations

import copy
import dataclasses

import torch

from .attention import packed_attention
from .kv_cache import append_kv, paged_attention, read_kv


class KVCache:
    """One layer's pages of keys and values (see ``append_kv``), in bfloat16
    or, `quantised`, in E4M3 with a power of two a row."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, *, quantised: bool = False, device=None):
        shape = (pages, kv_heads, page_size, head_dim)
        kind = torch.uint8 if quantised else torch.bfloat16
        self.k_pages, self.v_pages = (torch.zeros(shape, dtype=kind, device=device) for _ in range(2))
        self.k_scales = torch.zeros(shape[:3], dtype=torch.uint8, device=device) if quantised else None
        self.v_scales = torch.zeros_like(self.k_scales) if quantised else None

    def append(self, k, v, page_table, lengths, offsets=None) -> None:
        append_kv(k, v, self.k_pages, self.v_pages, page_table, lengths, offsets, k_scales=self.k_scales,
                  v_scales=self.v_scales)

    def read(self, page_table, offsets, rows: int):
        return read_kv(self.k_pages, self.v_pages, page_table, offsets, rows, k_scales=self.k_scales, v_scales=self.v_scales)

    def attend(self, q, page_table, lengths, *, scale=None):
        return paged_attention(q, self.k_pages, self.v_pages, page_table, lengths, k_scales=self.k_scales,
                               v_scales=self.v_scales, scale=scale)


class _After:
    """The field ``AttentionBatch.after``: what was given, else made of the
    lengths as they are when it is asked for.  What was made so is not taken as
    given where it is handed on, as dataclasses.replace does."""

    def __get__(self, batch, owner=None):
        if batch is None:
            return None  # the field's default
        if batch._given is not None or batch.offsets is not None:
            return batch._given
        made = batch._tokens()
        made.of_lengths = True
        return made

    def __set__(self, batch, value):
        batch._given = None if getattr(value, "of_lengths", False) else value


@dataclasses.dataclass
class AttentionBatch:
    """Which rows of a step are whose, the same for every layer.

    offsets int32 [sequences + 1]: packed rows (None with a page_table: one
    new token a sequence).  With a cache: page_table and lengths as for
    ``append_kv``.  Packed rows then attend to each other alone, so that their sequences
    hold nothing yet (a step with a length that is not 0 gives NaN), or to all that
    their sequences hold with them, by key_offsets, the offsets of lengths + new
    tokens, and keys, their last one, as a number.
    after: what single tokens' sequences hold with them, lengths + 1 where it is not
    given: as lengths are when a step runs, a captured one too.  A slot of single tokens is idle,
    and its attention 0, where it holds nothing and has no first page (a negative one)."""

    offsets: torch.Tensor | None = None
    page_table: torch.Tensor | None = None
    lengths: torch.Tensor | None = None
    key_offsets: torch.Tensor | None = None
    keys: int | None = None
    after: torch.Tensor | None = _After()

    def __post_init__(self):
        self._refused = False
        if (self.page_table is None) != (self.lengths is None):
            raise ValueError("page_table and lengths are given together")
        if self.page_table is None and (self.offsets is None or self.key_offsets is not None):
            raise ValueError("a batch without a cache has offsets, and no key_offsets")
        if (self.key_offsets is None) != (self.keys is None) or (self.key_offsets is not None and self.offsets is None):
            raise ValueError("key_offsets and keys are given together, with offsets")

    def _tokens(self) -> torch.Tensor:
        table = self.page_table
        if table.shape[:1] == self.lengths.shape and table.shape[1] > 0:
            return self.lengths + (table[:, 0] >= 0)
        return self.lengths + 1  # tables that do not fit are refused where they are used

    def refuse(self, x: torch.Tensor) -> torch.Tensor:
        """x; NaN in its place where the batch has packed rows leave out tokens that
        their sequences hold.  Decided on the device: the lengths are there."""
        if self._refused or self.offsets is None or self.page_table is None or self.key_offsets is not None:
            return x
        return torch.where(self.lengths.any(), float("nan"), x)

    def for_step(self) -> "AttentionBatch":
        """The same for all layers of a step: `after` made once, refused (or not) already."""
        if self.offsets is None and self._given is not None or self.page_table is None:
            return self
        step = copy.copy(self)
        if self.offsets is None:
            step.after = self._tokens()
        step._refused = True
        return step


class _ReadBack(torch.autograd.Function):
    """Keys and values as a cache gives them for those that were written to it:
    no gradient finds the way back, so that a backward pass raises."""

    @staticmethod
    def forward(ctx, k_new, v_new, k, v):
        return k.view_as(k), v.view_as(v)

    @staticmethod
    def backward(ctx, d_k, d_v):
        raise RuntimeError("keys and values that went through a cache have no gradient")


class SelfAttention(torch.nn.Module):
    """``o_proj(attention(qkv_proj(x)))``.  qkv_proj holds the query heads' rows,
    then the key heads', then the values'; both are any module from bfloat16
    rows to bfloat16 rows (nn.Linear, Int4Linear, BlockFP8Linear).  cache: a
    KVCache, for batches with a page table; what is read from it has no gradient, and a
    backward pass through it raises."""

    takes_batch = True

    def __init__(self, hidden_size: int, heads: int, kv_heads: int, head_dim: int | None = None, *, causal: bool = True,
                 scale: float | None = None, device=None):
        super().__init__()
        head_dim = hidden_size // heads if head_dim is None else head_dim
        if heads % kv_heads:
            raise ValueError(f"{heads} query heads are not a multiple of {kv_heads} key heads")
        width = (heads + 2 * kv_heads) * head_dim
        self.qkv_proj = torch.nn.Linear(hidden_size, width, bias=False, device=device, dtype=torch.bfloat16)
        self.o_proj = torch.nn.Linear(heads * head_dim, hidden_size, bias=False, device=device, dtype=torch.bfloat16)
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.causal, self.scale = causal, scale
        self.cache: KVCache | None = None

    def forward(self, x: torch.Tensor, batch: AttentionBatch | None = None) -> torch.Tensor:
        """x [..., hidden].  batch None: each x[i] of a [sequences, length,
        hidden] tensor is a sequence, or all of [length, hidden]."""
        lead = x.shape[:-1]
        rows = self.qkv_proj(x).reshape(-1, self.heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = rows.split([self.heads, self.kv_heads, self.kv_heads], 1)
        if batch is None:
            offsets = None
            if len(lead) > 1 and rows.shape[0]:
                offsets = torch.arange(0, rows.shape[0] + 1, lead[-1], dtype=torch.int32, device=x.device)
            out = packed_attention(q, k, v, offsets, causal=self.causal, scale=self.scale)
        else:
            out = self._attend(q, k, v, batch)
        return self.o_proj(out.reshape(*lead, self.heads * self.head_dim))

    def _attend(self, q, k, v, batch):
        if batch.page_table is None:
            return packed_attention(q, k, v, batch.offsets, causal=self.causal, scale=self.scale)
        if self.cache is None:
            raise RuntimeError("a batch with a page table needs a cache")
        if not self.causal:
            raise RuntimeError("a cache is of causal attention")
        k = batch.refuse(k)
        self.cache.append(k, v, batch.page_table, batch.lengths, batch.offsets)
        if batch.offsets is None:
            return self.cache.attend(q, batch.page_table, batch.after, scale=self.scale)
        if batch.key_offsets is not None:
            k_new, v_new, (k, v) = k, v, self.cache.read(batch.page_table, batch.key_offsets, batch.keys)
            if torch.is_grad_enabled() and (k_new.requires_grad or v_new.requires_grad):
                k, v = _ReadBack.apply(k_new, v_new, k, v)
        return packed_attention(q, k, v, batch.offsets, batch.key_offsets, scale=self.scale)

    def to_int4(self, group_size: int = 64, symmetric: bool = False) -> "SelfAttention":
        """The served form: the same with 4-bit projections, and without a cache."""
        from .int4 import Int4Linear

        served = SelfAttention(1, self.heads, self.kv_heads, self.head_dim, causal=self.causal, scale=self.scale, device="meta")
        for name in ("qkv_proj", "o_proj"):
            setattr(served, name, Int4Linear.from_linear(getattr(self, name), group_size=group_size, symmetric=symmetric))
        return served
