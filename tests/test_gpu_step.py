"""A step's tables and its accepted path on the GPU: whole numbers, equal to the oracle's."""

import numpy as np
import pytest
import torch

from oracle import tree
from wavelet_amd import accept_tree, extend_tables

pytestmark = pytest.mark.gpu


def _dev(x, cuda, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x), dtype=dtype).to(cuda)


def _parents(rng, new, rows):
    p = np.full(rows, -1, np.int32)
    at = 0
    for n in new:
        for i in range(1, n):
            if at + i < rows:
                p[at + i] = rng.integers(max(0, i - 9), i)
        at += max(int(n), 0)
    return p


def _case(seed, batch, ctx, new, bs, width, spare, extra=0):
    rng = np.random.default_rng(seed)
    lens, new = rng.integers(ctx[0], ctx[1] + 1, batch), rng.integers(new[0], new[1] + 1, batch)
    held = np.minimum(-(-lens // bs) + rng.integers(0, 2, batch), width)
    ids = rng.permutation(int(held.sum()) + spare).astype(np.int32)
    bt = np.full((batch, width), -1, np.int32)
    at = 0
    for i, h in enumerate(held):
        bt[i, :h] = ids[at:at + h]
        at += h
    return rng, bt, held, lens, new, ids[at:]


def _run(cuda, bt, held, lens, new, free, taken, bs, rows, parents, nodes, what, row_pad=0):
    table = torch.full((len(bt), bt.shape[1] + row_pad), -7, dtype=torch.int32, device=cuda)
    table[:, :bt.shape[1]] = _dev(bt, cuda)
    state = [_dev(x, cuda) for x in (held, lens, new, free)]
    before = [x.clone() for x in state]
    m = extend_tables(table[:, :bt.shape[1]], *state, _dev([taken], cuda), bs, rows,
                      parents=None if parents is None else _dev(parents, cuda), max_nodes=nodes)
    want = tree.extend_tables(bt, held, lens, new, free, taken, bs, rows, parents=parents, max_nodes=nodes)
    np.testing.assert_array_equal(table[:, :bt.shape[1]].cpu(), want["block_table"], err_msg=what)
    assert (table[:, bt.shape[1]:] == -7).all()
    for name in ("context_lens", "cu_seqlens_q", "slot_mapping", "positions", "held_blocks"):
        np.testing.assert_array_equal(getattr(m, name).cpu(), want[name], err_msg=f"{what}: {name}")
    assert int(m.taken) == want["taken"] and int(m.refused) == want["refused"], what
    if nodes:
        np.testing.assert_array_equal(m.tree_mask.cpu(), want["tree_mask"], err_msg=what)
    for x, y in zip(state, before):
        assert torch.equal(x, y)
    return want


@pytest.mark.parametrize("seed,batch,ctx,new,bs,width,spare", [
    (0, 1, (0, 0), (1, 1), 16, 1, 1), (1, 5, (0, 200), (0, 40), 16, 20, 60), (2, 64, (500, 4096), (16, 16), 16, 262, 200),
    (3, 64, (0, 0), (300, 2000), 16, 126, 9000), (4, 700, (0, 900), (1, 1), 32, 40, 90), (5, 2048, (0, 64), (0, 3), 16, 6, 900),
    (6, 33, (0, 100), (0, 300), 48, 9, 70), (7, 1025, (1, 40), (3, 5), 64, 2, 400), (8, 3, (30000, 32000), (5000, 9000), 16, 2600, 1700)])
def test_tables(cuda, seed, batch, ctx, new, bs, width, spare):
    rng, bt, held, lens, n, free = _case(seed, batch, ctx, new, bs, width, spare)
    total = int(n.sum())
    for rows in {total, total + 65, max(total - 3, 0)}:
        _run(cuda, bt, held, lens, n, free, 0, bs, rows, None, 0, f"chains {rows}", row_pad=seed % 3)
    short = len(free) // 2
    w = _run(cuda, bt, held, lens, n, free, short, bs, total, None, 0, "half taken")
    assert (w["refused"] > 0) == (seed in (6, 8))  # the two whose sequences need more than is left


@pytest.mark.parametrize("seed,batch,new,nodes", [(0, 1, (1, 1), 64), (1, 64, (16, 16), 64), (2, 9, (0, 70), 128),
                                                  (3, 3, (200, 256), 256), (4, 300, (1, 40), 64), (5, 40, (100, 256), 256)])
def test_tree_tables(cuda, seed, batch, new, nodes):
    rng, bt, held, lens, n, free = _case(seed, batch, (0, 300), new, 16, 40, 1200)
    rows = int(n.sum()) + 5
    parents = _parents(rng, n, rows)
    parents[rng.integers(0, rows, rows // 10)] = 250  # no earlier node: follows the context
    parents[rng.integers(0, rows, rows // 10)] = -3
    _run(cuda, bt, held, lens, n, free, 3, 16, rows, parents, nodes, "trees")
    chain = np.concatenate([np.arange(-1, x - 1) for x in n] + [np.full(5, -1)]).astype(np.int32)
    _run(cuda, bt, held, lens, n, free, 3, 16, rows, chain, nodes, "chains as trees")


def test_tables_of_odd_values(cuda):
    """Negative lengths count as 0; more taken than there is, no free blocks, tables without a block for a token."""
    bt = np.array([[4, -1, -1], [-1, 7, -1], [9, 8, -1]], np.int32)
    held, lens, new = [1, 2, 2], [10, -5, 40], [3, 4, -2]
    free = np.array([1, 2], np.int32)
    w = _run(cuda, bt, held, lens, new, free, 5, 16, 9, None, 0, "odd")
    assert w["refused"] == 0 and (w["slot_mapping"][3:7] == -1).all()  # the second's first block is none
    _run(cuda, bt, held, lens, new, free[:0], 0, 16, 9, None, 0, "none free")
    _run(cuda, bt, held, lens, [2**31 - 1, 5, 2**31 - 1], free, 0, 16, 9, None, 0, "huge")


def test_tables_state_in_place_and_captured(cuda):
    """The state carried on in its own tensors, replay after replay, as the oracle carries it."""
    B, bs, rows = 6, 16, 32
    bt = torch.full((B, 12), -1, dtype=torch.int32, device=cuda)
    held, lens, taken = (torch.zeros(n, dtype=torch.int32, device=cuda) for n in (B, B, 1))
    new = _dev([3, 0, 5, 1, 16, 7], cuda)
    free = _dev(np.random.default_rng(0).permutation(20), cuda)

    def step(out=None):
        return extend_tables(bt, held, lens, new, free, taken, bs, rows, out=out)

    out = step()._replace(held_blocks=held, taken=taken)
    bt.fill_(-1)
    held.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out)
        lens.copy_(torch.where(out.context_lens > 0, out.context_lens, lens))
    h, l, t, table = np.zeros(B, int), np.zeros(B, int), 0, np.full((B, 12), -1)
    refused = 0
    for i in range(12):
        graph.replay()
        torch.cuda.synchronize()
        w = tree.extend_tables(table, h, l, new.cpu().numpy(), free.cpu().numpy(), t, bs, rows)
        for name in ("context_lens", "cu_seqlens_q", "slot_mapping", "positions", "held_blocks"):
            np.testing.assert_array_equal(getattr(out, name).cpu(), w[name], err_msg=f"replay {i}: {name}")
        np.testing.assert_array_equal(bt.cpu(), w["block_table"])
        assert int(taken) == w["taken"]
        h, t, table = w["held_blocks"], w["taken"], w["block_table"]
        l = np.where(w["context_lens"] > 0, w["context_lens"], l)
        refused += w["refused"]
    assert refused > 0


def test_tables_refusals(cuda):
    i = torch.zeros(2, dtype=torch.int32, device=cuda)
    bt = torch.zeros((2, 3), dtype=torch.int32, device=cuda)
    ok = dict(block_table=bt, held_blocks=i, seq_lens=i, new_lens=i, free_blocks=i, taken=i[:1], block_size=16, max_tokens=4)
    extend_tables(**ok)
    p = torch.zeros(4, dtype=torch.int32, device=cuda)
    for bad in (dict(block_table=bt.long()), dict(block_table=bt.t()), dict(block_table=bt[:0]), dict(held_blocks=i.long()),
                dict(seq_lens=i[:1]), dict(new_lens=i.cpu()), dict(taken=i), dict(block_size=0), dict(max_tokens=-1),
                dict(parents=p), dict(max_nodes=64), dict(parents=p, max_nodes=65), dict(parents=p, max_nodes=320),
                dict(parents=p[:3], max_nodes=64), dict(block_table=bt[:1].expand(2, 3)), dict(out=(i,))):
        with pytest.raises(ValueError):
            extend_tables(**{**ok, **bad})
    m = extend_tables(**ok)
    with pytest.raises(ValueError):
        extend_tables(**ok, out=m._replace(slot_mapping=m.slot_mapping[:2]))
    with pytest.raises(ValueError):
        extend_tables(**ok, out=m._replace(context_lens=i))  # also an input


# ---------------------------------------------------------------------------- acceptance

@pytest.mark.parametrize("seed,batch,new,depth", [(0, 1, (1, 1), 1), (1, 5, (0, 8), 3), (2, 256, (64, 64), 16),
                                                  (3, 33, (1, 130), 64), (4, 7, (250, 256), 64), (5, 1000, (2, 5), 8)])
def test_accept(cuda, seed, batch, new, depth):
    rng = np.random.default_rng(seed)
    n = rng.integers(new[0], new[1] + 1, batch)
    cu = np.concatenate([[0], np.cumsum(n)])
    rows = int(cu[-1])
    parents = _parents(rng, n, rows)
    if seed == 4:  # chains that agree: the depth limit ends them
        parents = np.concatenate([np.arange(-1, x - 1) for x in n]).astype(np.int32)
    draft, target = rng.integers(0, 1 if seed == 4 else 2, (2, rows)) + 2**40
    lens = rng.integers(0, 5000, batch)
    context = np.where(rng.random(batch) < 0.1, 0, lens + n)  # some refused
    args = [_dev(draft, cuda, torch.int64), _dev(parents, cuda), _dev(target, cuda, torch.int64), _dev(cu, cuda),
            _dev(lens, cuda), _dev(context, cuda)]
    got = accept_tree(*args, depth)
    want = tree.accept_tree(draft, parents, target, cu, lens, context, depth)
    for x, y in zip(got, want):
        np.testing.assert_array_equal(x.cpu(), y)
    # the lengths in place
    again = accept_tree(*args, depth, out=got._replace(seq_lens=args[4]))
    assert again.seq_lens is args[4]
    np.testing.assert_array_equal(args[4].cpu(), want[3])


def test_accept_without_rows_and_refusals(cuda):
    z, i = torch.zeros(0, dtype=torch.int64, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    cu = torch.zeros(3, dtype=torch.int32, device=cuda)
    got = accept_tree(z, z.int(), z, cu, i + 3, i + 3, 4)
    assert got.accepted.tolist() == [0, 0] and got.next_tokens.tolist() == [-1, -1] and got.seq_lens.tolist() == [3, 3]
    assert (got.path == -1).all()
    assert accept_tree(z, z.int(), z, cu[:1], i[:0], i[:0], 4).path.shape == (0, 4)
    # rows that there are not (a longer step's cu_seqlens_q): nodes past the last are none
    t = torch.tensor([5, 6, 7], device=cuda)
    got = accept_tree(t, torch.tensor([-1, 0, 1], dtype=torch.int32, device=cuda), t + 1, cu + 100 * i.new_tensor([0, 1, 2]),
                      i + 3, i + 9, 4)
    assert got.accepted.tolist() == [3, 0] and got.next_tokens.tolist() == [8, -1] and got.path[0].tolist() == [0, 1, 2, -1]
    for bad in ((z.int(), z.int(), z, cu, i, i, 4), (z, z, z, cu, i, i, 4), (z, z.int(), z, cu, i[:1], i, 4),
                (z, z.int(), z, cu, i, i, 0), (z, z.int(), z, cu, i, i, 65), (z, z.int(), z.cpu(), cu, i, i, 4)):
        with pytest.raises(ValueError):
            accept_tree(*bad)
