"""Steps that reach the length limit on the GPU: whole numbers, equal to the oracle's; and whole drafted steps."""

import numpy as np
import pytest
import torch

from kvcase import bits_of, check_attention
from oracle import paged, tree
from test_gpu_step import _case, _dev, _parents
from wavelet_amd import KVPool, extend_tables
from wavelet_amd.plan import TreeStep

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed,batch,ctx,new,bs,width,spare,nodes,limit", [
    (0, 1, (40, 40), (10, 10), 16, 4, 4, 0, 50), (1, 1, (41, 41), (10, 10), 16, 4, 4, 0, 50),
    (2, 40, (20, 60), (0, 12), 16, 5, 60, 64, 59), (3, 300, (0, 90), (1, 30), 32, 5, 900, 64, 90),
    (4, 64, (0, 900), (50, 120), 16, 70, 900, 0, 777), (5, 9, (0, 70), (100, 256), 48, 9, 90, 256, 201),
    (6, 5, (0, 30), (0, 9), 16, 4, 9, 0, 0), (7, 5, (0, 30), (0, 9), 16, 4, 9, 0, 2**31 - 1)])
def test_tables_up_to_a_limit(cuda, seed, batch, ctx, new, bs, width, spare, nodes, limit):
    rng, bt, held, lens, n, free = _case(seed, batch, ctx, new, bs, width, spare)
    rows = int(n.sum())
    parents = _parents(rng, n, rows) if nodes else None
    table = _dev(bt, cuda)
    m = extend_tables(table, *(_dev(x, cuda) for x in (held, lens, n, free)), _dev([1], cuda), bs, rows,
                      parents=None if parents is None else _dev(parents, cuda), max_nodes=nodes, max_seq_len=limit)
    want = tree.extend_tables(bt, held, lens, n, free, 1, bs, rows, parents=parents, max_nodes=nodes, max_seq_len=limit)
    np.testing.assert_array_equal(table.cpu(), want["block_table"])
    for name in ("context_lens", "cu_seqlens_q", "slot_mapping", "positions", "held_blocks"):
        np.testing.assert_array_equal(getattr(m, name).cpu(), want[name], err_msg=name)
    assert int(m.taken) == want["taken"] and int(m.refused) == want["refused"]
    if nodes:
        np.testing.assert_array_equal(m.tree_mask.cpu(), want["tree_mask"])
    past = (n > 0) & (lens + n > limit)
    assert past.any() == (seed not in (0, 7)) and (m.context_lens.cpu().numpy()[past] == 0).all()


def test_limit_refusals(cuda):
    i = torch.zeros(2, dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError, match="max_seq_len"):
        extend_tables(torch.zeros((2, 3), dtype=torch.int32, device=cuda), i, i, i, i, i[:1], 16, 4, max_seq_len=-1)


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
def test_steps_up_to_the_limit(cuda, kv):
    """A pool whose max_model_len ends inside a block: chains that agree take a sequence to the limit and not past
    it, every step's attention is the oracle's, and what settles the block manager can go on with."""
    hq, hkv, d, bs, limit, T = 4, 2, 64, 16, 90, 24
    pool = KVPool(1, 40, bs, hkv, d, kv, device=cuda, max_model_len=limit)
    for i, n in enumerate((60, 71)):
        pool.blocks.allocate(i, np.arange(n) + 1000 * i)
    c = pool.layers[0]
    c.append(*(torch.randn((131, hkv, d), device=cuda).to(torch.bfloat16) for _ in range(2)), torch.cat(
        [torch.from_numpy(pool.blocks.tables([i])[0][0].astype(np.int64)[np.arange(n) // bs] * bs + np.arange(n) % bs)
         for i, n in enumerate((60, 71))]).to(cuda))
    state = pool.lend([0, 1], 8)
    q, out = (torch.zeros((T, hq, d), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    k, v = (torch.zeros((T, hkv, d), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    new = torch.tensor([10, 10], dtype=torch.int32, device=cuda)
    parents = torch.cat([torch.arange(10) - 1, torch.arange(10) - 1, torch.full((4,), -1)]).to(cuda, torch.int32)
    tokens = torch.zeros(T, dtype=torch.int64, device=cuda)
    step = TreeStep(pool.layers, [q], [k], [v], [out], state, new, parents, tokens, tokens, d ** -0.5, 64, limit, 64)
    seen = []
    for i in range(4):
        for x in (q, k, v):
            x.normal_()
        lens = state.seq_lens.tolist()
        step.begin()
        step.run()
        context = step.maps.context_lens.tolist()
        assert context == [n + 10 if n + 10 <= limit else 0 for n in lens]
        if kv == "bf16":
            ref = tree.tree_gqa(paged.bf16_to_f32(bits_of(q)), *(paged.bf16_to_f32(x) for x in paged.logical_kv(
                bits_of(c.k), bits_of(c.v))), block_table=state.block_table.cpu().numpy(), seq_lens=context,
                cu_seqlens_q=step.maps.cu_seqlens_q.cpu().numpy(), tree_mask=step.maps.tree_mask.cpu().numpy(),
                scale=d ** -0.5)
            check_attention(paged.bf16_to_f32(bits_of(out))[:20], ref[:20], f"step {i}")
        step.finish()
        seen.append(int(step.maps.refused))
    assert seen == [0, 1, 1, 2] and state.seq_lens.tolist() == [90, 81]
    new.copy_(torch.tensor([0, 9]))  # a shorter tree still goes
    step.begin()
    step.run()
    step.finish()
    assert int(step.maps.refused) == 0 and state.seq_lens.tolist() == [90, 90]
    pool.settle(state)
    assert [pool.blocks.seq_len(i) for i in range(2)] == [90, 90]


def test_a_plans_own_limit(cuda):
    """max_seq_len of the plan below the pool's: refused, not attended wrongly."""
    pool = KVPool(1, 40, 16, 2, 64, device=cuda, max_model_len=300)
    pool.blocks.allocate(0, range(60))
    state = pool.lend([0], 8)
    z = lambda h: torch.zeros((8, h, 64), dtype=torch.bfloat16, device=cuda)  # noqa: E731
    i = torch.tensor([8], dtype=torch.int32, device=cuda)
    t = torch.zeros(8, dtype=torch.int64, device=cuda)
    for limit, refused in ((67, 1), (68, 0)):
        step = TreeStep(pool.layers, [z(4)], [z(2)], [z(2)], [z(4)], state, i, t.int() - 1, t, t, 0.125, 64, limit, 8)
        step.begin()
        assert int(step.maps.refused) == refused
