"""Loans taken back without a settlement, and loans that fail to be made (CPU)."""

import pytest

from wavelet_amd import BlockManager, KVPool


def _all(m, ids):
    return {s: (m.blocks_of(s), m.seq_len(s)) for s in ids}, m._ref.tolist(), m.num_free_blocks


def test_cancel_returns_every_block_and_keeps_the_host_side():
    m = BlockManager(40, 4)
    m.allocate("a", range(10))
    m.fork("a", "b")
    loan, cow = m.lend(["a", "b"], 6)
    assert len(cow) == 1
    before = _all(m, "ab")
    m.cancel(loan)
    now = _all(m, "ab")
    assert now[0] == before[0] and now[2] == before[2] + 6 and all(m.ref_count(b) == 0 for b in loan.blocks)
    for call in (lambda: m.cancel(loan), lambda: m.settle(loan, *m.tables("ab"), [3, 3])):
        with pytest.raises(ValueError, match="already"):
            call()
    assert _all(m, "ab") == now
    m.append_slots(["a", "b"], 9)
    for s in "ab":
        m.free(s)
    assert m.num_free_blocks == 40


@pytest.mark.parametrize("where", ["copy_blocks", "tensors"])
def test_a_loan_that_fails_leaves_nothing_lent(monkeypatch, where):
    pool = KVPool(2, 32, 16, 2, 64, device="cpu")
    pool.blocks.allocate(0, range(30))
    for s in (1, 2):
        pool.blocks.fork(0, s)
    before = _all(pool.blocks, [0, 1, 2])

    def fail(*a, **kw):
        raise RuntimeError("out of memory")

    if where == "copy_blocks":
        monkeypatch.setattr(pool, "copy_blocks", fail)
    else:
        monkeypatch.setattr("wavelet_amd.pool.StepState", fail)
    with pytest.raises(RuntimeError, match="out of memory"):
        pool.lend([0, 1, 2], 5)
    assert _all(pool.blocks, [0, 1, 2]) == before  # nor has a sequence a block that was never copied
    monkeypatch.undo()
    monkeypatch.setattr(pool, "copy_blocks", lambda pairs: None)
    state = pool.lend([0, 1, 2], 5)
    assert state.seq_lens.tolist() == [30] * 3


def test_pool_cancel(monkeypatch):
    pool = KVPool(2, 32, 16, 2, 64, device="cpu", max_model_len=160)
    pool.blocks.allocate(0, range(30))
    state = pool.lend([0], 5)
    state.seq_lens.numpy()[:] = 200  # what no settlement takes
    state.held_blocks.numpy()[:] = 7
    state.block_table.numpy()[0, 2:7] = state.free_blocks.numpy()
    with pytest.raises(ValueError):
        pool.settle(state)
    pool.cancel(state)
    assert pool.blocks.num_free_blocks == 30 and pool.blocks.seq_len(0) == 30
    pool.blocks.free(0)
    pool.sleep()
