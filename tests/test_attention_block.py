"""Batches that AttentionBlock refuses, whole: what was set before stays.  No kernel is launched here."""
import numpy as np
import pytest

pytest.importorskip("torch")

from decoder_stack import AttentionBlock


def test_batches_that_do_not_fit_the_block_are_refused():
    block = AttentionBlock(heads=2, kv_heads=1, head_dim=64, hidden=64, sequences=3, max_tokens=8, pages=9, pages_per_sequence=3, page_size=16, device="cpu")
    table = np.arange(9).reshape(3, 3)
    block.set_batch(table, [3, 20, 5], [0, 2, 2, 7], tokens=8)
    was = [t.clone() for t in (block.page_table, block.lengths, block.starts, block.positions)]
    assert block.tokens == 8 and block.positions.tolist() == [1, 2, 0, 1, 2, 3, 4, 0]
    for bad in (dict(page_table=[0, 1, 2]),  # (one sequence's pages would be those of all)
                dict(page_table=table[:1]), dict(page_table=table[:, :2]), dict(lengths=[3]), dict(lengths=[3, 20, 5, 1]), dict(starts=[0, 2, 7]),
                dict(starts=[0, 2, 1, 7]), dict(starts=[-1, 2, 2, 7]), dict(starts=[0, 2, 2, 9]), dict(tokens=6), dict(tokens=0), dict(tokens=9),
                dict(starts=[0, 2, 2, 9], tokens=None), dict(starts=[0, 0, 0, 0], tokens=None)):
        with pytest.raises(ValueError):
            block.set_batch(**dict(dict(page_table=table, lengths=[3, 20, 5], starts=[0, 2, 2, 7], tokens=8), **bad))
        assert block.tokens == 8 and all((a == b).all() for a, b in zip(was, (block.page_table, block.lengths, block.starts, block.positions)))


def test_a_block_of_one_sequence_takes_its_pages_as_a_row():
    block = AttentionBlock(heads=2, kv_heads=1, head_dim=64, hidden=64, max_tokens=4, pages=3, page_size=16, device="cpu")
    block.set_batch([2, 0, 1], [20], [0, 4])
    assert block.page_table.tolist() == [[2, 0, 1]] and block.positions.tolist() == [16, 17, 18, 19]
