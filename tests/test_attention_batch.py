"""CPU tests of AttentionBatch: what a step takes from it."""

from __future__ import annotations

import dataclasses

from conftest import pkg


def single(**changes):
    import torch

    table = torch.zeros(3, 2, dtype=torch.int32)
    return pkg().AttentionBatch(**{**dict(page_table=table, lengths=torch.tensor([4, 0, 9], dtype=torch.int32)), **changes})


def test_after_follows_the_lengths():
    """In place, by assignment, and in a copy with other lengths."""
    import torch

    batch = single()
    assert batch.after.tolist() == [5, 1, 10]
    batch.lengths += 1
    assert batch.after.tolist() == [6, 2, 11] and batch.for_step().after.tolist() == [6, 2, 11]
    batch.lengths = torch.tensor([7, 7, 7], dtype=torch.int32)
    assert batch.after.tolist() == [8, 8, 8]
    other = dataclasses.replace(batch, lengths=batch.lengths + 5)
    assert other.after.tolist() == [13, 13, 13]
    other.lengths += 1
    assert other.after.tolist() == [14, 14, 14]
    taken = single(after=batch.after)  # another batch's, made there
    assert taken.after.tolist() == [5, 1, 10]


def test_an_own_after_stays():
    import torch

    own = torch.tensor([1, 2, 3], dtype=torch.int32)
    batch = single(after=own)
    batch.lengths += 1
    assert batch.after is own and batch.for_step() is batch
    assert dataclasses.replace(batch, lengths=batch.lengths + 1).after is own


def test_packed_rows_have_none():
    import torch

    offsets = torch.tensor([0, 2, 5], dtype=torch.int32)
    batch = pkg().AttentionBatch(offsets)
    assert batch.after is None and batch.for_step() is batch


def test_idle_slots_hold_nothing():
    """A slot without a first page keeps its length: 0 where it is idle, a token without a page where it is not."""
    import torch

    table = torch.tensor([[3, -1], [-1, -1], [-1, 2]], dtype=torch.int32)
    batch = single(page_table=table, lengths=torch.tensor([4, 0, 9], dtype=torch.int32))
    assert batch.after.tolist() == [5, 0, 9] and batch.for_step().after.tolist() == [5, 0, 9]
    assert single(page_table=table[:, :0]).after.tolist() == [5, 1, 10]


def test_packed_rows_of_sequences_that_hold_tokens_are_refused():
    """Without key_offsets: NaN in place of what a step works on, once a step."""
    import torch

    def ints(*values):
        return torch.tensor(values, dtype=torch.int32)

    x, table = torch.arange(20.0).view(10, 2), torch.zeros(4, 2, dtype=torch.int32)
    batch = pkg().AttentionBatch(ints(1, 3, 3, 6, 8), table, ints(0, 5, 2, 0))
    assert bool(batch.refuse(x).isnan().all())
    step = batch.for_step()
    assert step.refuse(x) is x and step.lengths is batch.lengths and step.after is None
    batch.lengths.zero_()
    assert torch.equal(batch.refuse(x), x)
    for other in (pkg().AttentionBatch(ints(1, 3, 3, 6, 8), table, ints(0, 5, 2, 0), ints(1, 3, 8, 13, 15), 15),
                  pkg().AttentionBatch(ints(0, 3)), single()):
        assert other.refuse(x) is x


def test_blocks_without_attention_do_not_see_the_batch():
    """Not even one that attention would refuse."""
    import torch

    class Same(torch.nn.Module):
        mlp, eps, norm_weight = None, 1e-5, None

        def forward(self, residual, normed=None, next_weight=None, batch=None):
            return residual, normed

    table, ints = torch.zeros(1, 2, dtype=torch.int32), torch.tensor([0, 4], dtype=torch.int32)
    x = torch.ones(4, 8)
    assert pkg().run_blocks([Same()], x, None, pkg().AttentionBatch(ints, table, ints[1:]))[0] is x
