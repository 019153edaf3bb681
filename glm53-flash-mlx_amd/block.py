"""A feed-forward block around the package's feed-forwards: norm in front,
norm, gate and residual scale behind, the next block's input norm in the same
pass."""

from __future__ import annotations

import torch

from .norms import residual_norm, rms_norm


class FeedForwardBlock(torch.nn.Module):
    """``residual + scale * gate * post_norm(mlp(norm(residual)))``.

    mlp: any module that takes normalised bfloat16 [..., hidden] (GatedMLP,
    Int4MLP, ClampedMLP, PackedFP8MoE, SortedGroupedFP8MoE, ...) and returns
    bfloat16 or float32.  The residual stream may be bfloat16 or float32.  gate: a learned value a channel;
    forward's own `gate` (a token's, a sequence's: see residual_norm) stands in
    for it."""

    def __init__(self, mlp: torch.nn.Module, hidden_size: int, *, eps: float = 1e-6, post_norm: bool = True,
                 gate: bool = False, residual_scale: float = 1.0, device=None, dtype: torch.dtype = torch.bfloat16):
        super().__init__()

        def ones():
            return torch.nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype))

        self.mlp = mlp
        self.norm_weight = ones()
        self.post_weight = ones() if post_norm else None
        self.gate = ones() if gate else None
        self.eps, self.residual_scale = float(eps), float(residual_scale)

    def forward(self, residual: torch.Tensor, normed: torch.Tensor | None = None,
                next_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None):
        """``(new residual, normed)``.  normed: this block's input where the
        block before has made it; next_weight: the norm weight that the
        returned `normed` is made with (None: no such norm, returns None)."""
        if normed is None:
            normed = rms_norm(residual, self.norm_weight, self.eps, dtype=torch.bfloat16)
        elif normed.dtype is not torch.bfloat16:  # the block before returned another type
            normed = normed.to(torch.bfloat16)
        return residual_norm(residual, self.mlp(normed), post_weight=self.post_weight,
                             gate=self.gate if gate is None else gate, scale=self.residual_scale,
                             next_weight=next_weight, eps=self.eps)


def run_blocks(blocks, residual: torch.Tensor, final_weight: torch.Tensor | None = None):
    """The blocks in turn, each norm between two made by the pass that ends
    the first: ``(residual, residual normed with final_weight or None)``."""
    blocks = list(blocks)
    if not blocks:
        raise ValueError("run_blocks needs a block")
    normed = None
    for block, after in zip(blocks, blocks[1:] + [None]):
        weight = final_weight if after is None else after.norm_weight
        if after is not None and after.eps != block.eps:
            raise ValueError("blocks in a run share one eps")
        residual, normed = block(residual, normed, weight)
    return residual, normed
