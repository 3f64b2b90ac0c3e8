"""No loan settles past max_model_len, and a refused settlement changes nothing (CPU)."""

import pytest

from wavelet_amd import BlockManager


def test_settle_refuses_lengths_past_the_limit():
    m = BlockManager(20, 16, max_model_len=40)
    m.allocate("a", range(30))
    loan, _ = m.lend(["a"], 2)
    bt, _ = m.tables(["a"], 4)
    bt[0, 2] = loan.blocks[0]
    for length in (41, 48):
        with pytest.raises(ValueError, match="max_model_len"):
            m.settle(loan, bt, [3], [length])
        assert m.seq_len("a") == 30 and len(m.blocks_of("a")) == 2 and m.num_free_blocks == 20 - 4
    m.settle(loan, bt, [3], [40])
    assert m.seq_len("a") == 40 and m.num_free_blocks == 20 - 3
    with pytest.raises(ValueError, match="max_model_len"):
        m.append_slots(["a"])
