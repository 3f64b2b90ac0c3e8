"""A loan is settled once, whatever was lent since (CPU)."""

import numpy as np
import pytest

from wavelet_amd import BlockManager


def _state(m):
    return ({s: (m.blocks_of(s), m.seq_len(s)) for s in ("a", "b")}, m._ref.tolist(), sorted(m._free), m.num_free_blocks)


def test_an_old_loan_of_sequences_lent_again():
    m = BlockManager(20, 4)
    m.allocate("a", range(10))
    m.allocate("b", range(100, 108))
    old, _ = m.lend(["a", "b"], 3)
    bt, lens = m.tables(["a", "b"], 6)
    bt[0, 3] = old.blocks[0]
    m.settle(old, bt, [4, 2], [13, 8])  # "a" keeps a lent block
    new, _ = m.lend(["a", "b"], 2)
    before = _state(m)
    with pytest.raises(ValueError, match="already"):
        m.settle(old, bt, [4, 2], [13, 8])
    assert _state(m) == before
    with pytest.raises(ValueError, match="device"):  # still lent
        m.append_slots(["a"])
    bt, lens = m.tables(["a", "b"], 6)
    m.settle(new, bt, [4, 2], lens)
    for s in ("a", "b"):
        m.free(s)
    assert m.num_free_blocks == 20 and (m._ref == 0).all()


def test_a_loan_to_no_sequence():
    m = BlockManager(8, 4)
    loan, _ = m.lend([], 3)
    assert m.num_free_blocks == 5
    nothing = (np.zeros((0, 1)), [], [])
    m.settle(loan, *nothing)
    assert m.num_free_blocks == 8
    with pytest.raises(ValueError, match="already"):
        m.settle(loan, *nothing)
    assert m.num_free_blocks == 8 and (m._ref == 0).all()


def test_a_loan_of_another_manager():
    m, other = BlockManager(8, 4), BlockManager(8, 4)
    for x in (m, other):
        x.allocate("a", range(6))
    mine, _ = m.lend(["a"], 2)
    theirs, _ = other.lend(["a"], 2)
    bt, lens = m.tables(["a"])
    with pytest.raises(ValueError):
        m.settle(theirs, bt, [2], lens)
    m.settle(mine, bt, [2], lens)
