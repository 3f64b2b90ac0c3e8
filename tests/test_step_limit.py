"""The length limit of steps whose tokens the host does not count (CPU): what a loan carries, and the oracle's rule."""

import numpy as np
import pytest

from oracle import tree
from test_tree_oracle import P, host_only
from wavelet_amd import BlockManager, KVPool, _lib


def test_a_loan_carries_the_pools_limit():
    for limit in (None, 50):
        pool = KVPool(1, 16, 16, 2, 64, device="cpu", max_model_len=limit)
        pool.blocks.allocate(0, range(30))
        assert pool.lend([0], 3).max_seq_len == limit


def test_the_oracle_refuses_what_the_block_manager_does():
    """A limit that is no multiple of the block size: room in the last block is not room in the sequence."""
    m = BlockManager(16, 16, max_model_len=50)
    for i, n in enumerate((41, 42, 50)):
        m.allocate(i, np.arange(n) + 100 * i)
    bt, lens = m.tables([0, 1, 2])
    held = [len(m.blocks_of(i)) for i in range(3)]
    t = tree.extend_tables(bt, held, lens, [9, 9, 0], np.arange(10), 0, 16, 18, max_seq_len=50)
    assert t["context_lens"].tolist() == [50, 0, 50] and t["refused"] == 1
    m.append_slots([0], 9)
    with pytest.raises(ValueError, match="max_model_len"):
        m.append_slots([1], 9)


@host_only
@pytest.mark.parametrize("kw", [dict(limit=-1), dict(batch=0), dict(words=5), dict(bt=None), dict(context=2 * P)])
def test_limited_tables_refusals(kw):
    a = dict(bt=P, stride=8, width=8, held=P, lens=2 * P, new=3 * P, batch=2, bs=16, free=P, nfree=4, taken=P, rows=8,
             limit=100, parents=P, words=1, held_out=P, taken_out=P, context=4 * P, cu=P, slots=P, pos=P, mask=P, refused=P,
             stream=None)
    a.update(kw)
    assert _lib.load().wkv_extend_tables_limited(*a.values()) == _lib.WKV_ERR_INVALID
