"""Blocks lent to the device (CPU): the block manager's side of steps whose token counts it does not know."""

import numpy as np
import pytest

from oracle import tree
from wavelet_amd import BlockManager, KVPool


def _manager(blocks=40, bs=4):
    m = BlockManager(blocks, bs)
    m.allocate("a", range(10))   # three blocks, the last partly filled
    m.allocate("b", range(100, 108))  # two, full
    m.share_prefix("a", ["c", "d"], None)
    return m


def test_lend_makes_partly_filled_blocks_private_and_counts_first():
    m = _manager()
    free, shared = m.num_free_blocks, m.blocks_of("a")
    loan, cow = m.lend(["a", "b", "c", "d"], 6)
    # of the three holders of the shared last block two get copies; the third is then alone
    assert [src for src, _ in cow] == [shared[2]] * 2 and m.num_free_blocks == free - 6 - 2
    last = [m.blocks_of(s)[2] for s in "acd"]
    assert len(set(last)) == 3 and all(m.ref_count(b) == 1 for b in last)
    assert all(m.blocks_of(s)[:2] == shared[:2] for s in "acd") and m.ref_count(shared[0]) == 3
    assert len(set(loan.blocks)) == 6 and all(m.ref_count(b) == 1 for b in loan.blocks)


@pytest.mark.parametrize("bad", [dict(num_blocks=-1), dict(seq_ids=["a", "a"]), dict(num_blocks=1000), dict(num_blocks=35)])
def test_lend_refuses_and_changes_nothing(bad):
    m = _manager(blocks=40)
    tables, free = [m.blocks_of(s) for s in "abcd"], m.num_free_blocks  # 35 free, two of them for copies
    with pytest.raises((ValueError, MemoryError)):
        m.lend(**{"seq_ids": ["a", "b", "c", "d"], "num_blocks": 2, **bad})
    assert [m.blocks_of(s) for s in "abcd"] == tables and m.num_free_blocks == free
    m.lend(["a", "b", "c", "d"], 33)


def test_lent_sequences_are_the_devices_until_settled():
    m = _manager()
    loan, _ = m.lend(["a", "b"], 4)
    for call in (lambda: m.append_slots(["a"]), lambda: m.free("b"), lambda: m.fork("a", "e"), lambda: m.lend(["b"], 1),
                 lambda: m.blocks_needed(["a"])):
        with pytest.raises(ValueError, match="device"):
            call()
    m.append_slots(["c"])  # the others are not
    bt, lens = m.tables(["a", "b"])
    m.settle(loan, bt, [3, 2], lens)
    m.append_slots(["a"])
    with pytest.raises(ValueError, match="already"):
        m.settle(loan, bt, [3, 2], lens)


@pytest.mark.parametrize("seed", range(4))
def test_steps_on_the_device_and_back(seed):
    """Random steps by the oracle of extend_tables, some tokens rejected: what settles is as if the host had
    appended the tokens kept, and every block is held or free."""
    rng = np.random.default_rng(seed)
    m = _manager(60)
    ids = list("abcd")
    loan, _ = m.lend(ids, 30)
    held = np.array([len(m.blocks_of(s)) for s in ids], np.int32)
    bt, lens = m.tables(ids, 20)
    taken = 0
    for _ in range(5):
        new = rng.integers(0, 7, 4)
        t = tree.extend_tables(bt, held, lens, new, np.array(loan.blocks), taken, 4, int(new.sum()))
        bt, held, taken = t["block_table"], t["held_blocks"], t["taken"]
        lens = lens + np.where(new > 0, rng.integers(0, new + 1), 0).astype(np.int32)
    m.settle(loan, bt, held, lens)
    for i, s in enumerate(ids):
        assert m.seq_len(s) == lens[i]
        assert m.blocks_of(s) == bt[i, :max(-(-int(lens[i]) // 4), [3, 2, 3, 3][i])].tolist()
    owned = {b for s in ids for b in m.blocks_of(s)}
    assert m.num_free_blocks == 60 - len(owned)
    m.append_slots(ids, 3)
    for s in ids:
        m.free(s)
    assert m.num_free_blocks == 60


def test_settle_refuses_foreign_tables_and_changes_nothing():
    m = _manager()
    loan, _ = m.lend(["a", "b"], 4)
    bt, lens = m.tables(["a", "b"], 6)
    bt[0, 3], bt[1, 2] = loan.blocks[0], loan.blocks[1]
    held, lens = np.array([4, 3]), lens + 2
    foreign = m.blocks_of("c")[0]
    for at, value in (((0, 3), foreign), ((0, 3), -1), ((0, 0), loan.blocks[3]), ((1, 2), loan.blocks[0])):
        x = bt.copy()
        x[at] = value
        with pytest.raises(ValueError):
            m.settle(loan, x, held, lens)
    for h, n in (([7, 3], lens), ([2, 3], lens), (held, [17, 8]), (held, [9, 10]), ([4], lens)):
        with pytest.raises(ValueError):
            m.settle(loan, bt, np.array(h), np.array(n))
    m.settle(loan, bt, held, lens)
    assert m.seq_len("a") == 12 and m.blocks_of("b")[2] == loan.blocks[1]
    assert m.blocks_of("a") == bt[0, :3].tolist() and m.ref_count(loan.blocks[0]) == 0  # 12 tokens fill three blocks


def test_pool_lends_and_settles():
    pool = KVPool(2, 32, 16, 2, 64, device="cpu", max_model_len=160)
    pool.blocks.allocate(0, range(30))
    pool.blocks.allocate(1, range(16))
    s = pool.lend([0, 1], 5)
    assert tuple(s.block_table.shape) == (2, 10) and s.held_blocks.tolist() == [2, 1] and s.seq_lens.tolist() == [30, 16]
    assert s.free_blocks.tolist() == s.loan.blocks and int(s.taken) == 0 and s.block_size == 16
    t = tree.extend_tables(s.block_table.numpy(), s.held_blocks.numpy(), s.seq_lens.numpy(), [5, 4],
                           s.free_blocks.numpy(), 0, 16, 9)
    s.block_table.numpy()[:] = t["block_table"]
    s.held_blocks.numpy()[:] = t["held_blocks"]
    s.seq_lens.numpy()[:] = [33, 16]
    pool.settle(s)
    assert pool.blocks.seq_len(0) == 33 and len(pool.blocks.blocks_of(0)) == 3 and len(pool.blocks.blocks_of(1)) == 1
    assert pool.blocks.num_free_blocks == 32 - 3  # the prompts' first block is one
    for bad in (dict(seq_ids=[]), dict(seq_ids=[0], width=2)):
        with pytest.raises(ValueError):
            pool.lend(**{"num_blocks": 1, **bad})
    assert pool.blocks.num_free_blocks == 32 - 3
    for sid in (0, 1):
        pool.blocks.free(sid)
    pool.sleep()
    pool.blocks.allocate(2, range(5))
    with pytest.raises(RuntimeError, match="asleep"):
        pool.lend([2], 1)
    pool.blocks.append_slots([2])  # nothing is lent
