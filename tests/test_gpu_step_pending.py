"""The token that a sequence goes on with: kept where a step accepts nothing of it, on the GPU."""

import numpy as np
import pytest
import torch

from oracle import tree
from test_gpu_step import _dev, _parents
from wavelet_amd import KVPool, accept_tree
from wavelet_amd.plan import TreeStep

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [1, 5, 257])
def test_pending_tokens(cuda, batch):
    rng = np.random.default_rng(batch)
    n = rng.integers(0, 9, batch)
    n[0] = 3
    cu = np.concatenate([[0], np.cumsum(n)])
    parents = _parents(rng, n, int(cu[-1]))
    draft, target = rng.integers(0, 2, (2, int(cu[-1]))) + 2**40
    lens = rng.integers(0, 99, batch)
    context = np.where(rng.random(batch) < 0.3, 0, lens + n)
    was = rng.integers(0, 1000, batch)
    pending = _dev(was, cuda, torch.int64)
    got = accept_tree(*(_dev(x, cuda, t) for x, t in ((draft, torch.int64), (parents, torch.int32), (target, torch.int64),
                                                      (cu, torch.int32), (lens, torch.int32), (context, torch.int32))), 4,
                      pending=pending)
    acc, path, nxt, after = tree.accept_tree(draft, parents, target, cu, lens, context, 4)
    for x, y in zip((*got, pending), (acc, path, nxt, after, np.where(acc > 0, nxt, was))):
        np.testing.assert_array_equal(x.cpu(), y)


def test_pending_refusals(cuda):
    z, i = torch.zeros(3, dtype=torch.int64, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, 1, 3], dtype=torch.int32, device=cuda)
    for bad in (i, z, z[:2].cpu(), torch.zeros(4, dtype=torch.int64, device=cuda)[::2]):
        with pytest.raises(ValueError, match="pending"):
            accept_tree(z, z.int() - 1, z, cu, i, i, 4, pending=bad)


class Model:
    """A sequence's text is a rule of its tokens: next(x) = 3 x + 1 mod 1000; drafts are right or wrong at will."""

    @staticmethod
    def next(x):
        return (3 * x + 1) % 1000

    def text(self, first, n):
        out = [first]
        while len(out) < n:
            out.append(self.next(out[-1]))
        return out


@pytest.mark.parametrize("captured", [False, True])
def test_refused_and_paused_sequences_go_on(cuda, captured):
    """Three sequences, of which one is refused (no free block) and one paused now and then: every step's first
    nodes are state.next_tokens, and what each sequence accepts, step by step, is its text without a gap."""
    model, first = Model(), [7, 100, 555]
    pool = KVPool(1, 12, 16, 2, 64, device=cuda)
    for i, n in enumerate((14, 30, 31)):
        pool.blocks.allocate(i, np.arange(n) + 1000 * i)
    state = pool.lend([0, 1, 2], 4)
    assert state.next_tokens.tolist() == [-1] * 3
    state.next_tokens.copy_(torch.tensor(first))
    T, new = 12, torch.zeros(3, dtype=torch.int32, device=cuda)
    z = lambda h: torch.zeros((T, h, 64), dtype=torch.bfloat16, device=cuda)  # noqa: E731
    parents = torch.full((T,), -1, dtype=torch.int32, device=cuda)
    draft, target = (torch.zeros(T, dtype=torch.int64, device=cuda) for _ in range(2))
    step = TreeStep(pool.layers, [z(4)], [z(2)], [z(2)], [z(4)], state, new, parents, draft, target, 0.125, 64, 192, 8)
    graph = torch.cuda.CUDAGraph()
    if captured:
        for call in (step.begin, step.run, step.finish):  # a step of nothing
            call()
        assert state.next_tokens.tolist() == first
        with torch.cuda.graph(graph):
            step.begin()
            step.run()
            step.finish()
    texts, refused = [[], [], []], 0
    for i, lens in enumerate(([4, 4, 4], [0, 3, 2], [4, 0, 4], [1, 4, 4], [4, 4, 4], [4, 4, 4], [4, 4, 4], [0, 1, 1],
                              [4, 4, 4], [4, 4, 4], [2, 2, 2])):
        nodes, par, want = [], [], []
        for s, n in zip(state.next_tokens.tolist(), lens):
            chain = model.text(s, n) if n else []
            if n > 2 and i % 2:
                chain[2] = 999999  # a wrong draft
            nodes += chain
            par += list(range(-1, n - 1))
            want += [model.next(x) for x in chain]
        for dst, x, fill in ((draft, nodes, 0), (target, want, 0), (parents, par, -1)):
            dst.copy_(torch.tensor(x + [fill] * (T - len(x))))
        new.copy_(torch.tensor(lens))
        if captured:
            graph.replay()
        else:
            step.begin()
            step.run()
            step.finish()
        torch.cuda.synchronize()
        refused += int(step.maps.refused)
        cu, path = step.maps.cu_seqlens_q.tolist(), step.accepted.path.tolist()
        for b, n in enumerate(step.accepted.accepted.tolist()):
            texts[b] += [nodes[cu[b] + j] for j in path[b][:n]]
    assert refused > 0 and min(map(len, texts)) > 4
    for b in range(3):
        assert texts[b] == model.text(first[b], len(texts[b]))
        assert state.next_tokens[b] == model.text(first[b], len(texts[b]) + 1)[-1]
        assert int(state.seq_lens[b]) == (14, 30, 31)[b] + len(texts[b])


def test_pending_is_no_other_result(cuda):
    z, i = torch.zeros(3, dtype=torch.int64, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, 1, 3], dtype=torch.int32, device=cuda)
    got = accept_tree(z, z.int() - 1, z, cu, i, i, 4)
    with pytest.raises(ValueError, match="pending"):
        accept_tree(z, z.int() - 1, z, cu, i, i, 4, pending=got.next_tokens, out=got)
