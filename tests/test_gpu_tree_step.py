"""Steps of drafted tokens as a program runs them: blocks lent by the pool, tables, rotation, append, tree
attention of every layer, the accepted path and its move, several steps in a row, against the oracle.

Whole numbers and cache contents are the oracle's bit for bit (the keys appended are the rotated ones
that the step leaves in its buffer); rotations and attention as in their own tests: a rotated bf16
value is within 2^-8 of the exact one, relative to the pair's length, attention as for kvcase.check_attention.
"""

import numpy as np
import pytest
import torch

from kvcase import bits_of, check_attention
from oracle import fp8, paged, tree
from wavelet_amd import KVPool, rotary_frequencies
from wavelet_amd.plan import TreeStep

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
LAYERS, HQ, HKV, D, BS = 2, 8, 2, 64, 16
PROMPTS = (40, 3, 16, 640)
T, NODES, DEPTH = 96, 64, 8


class Program:
    """A pool with four prompts (the first shared by a fork), their blocks lent, and a TreeStep over it."""

    def __init__(self, cuda, kv):
        self.pool = KVPool(LAYERS, 120, BS, HKV, D, kv, device=cuda, max_model_len=900)
        b = self.pool.blocks
        for i, n in enumerate(PROMPTS):
            b.allocate(i, np.arange(n) + 1000 * i)
        b.fork(0, "fork")
        self.ids = [0, 1, 2, 3, "fork"]
        gen = torch.Generator(device=cuda).manual_seed(1)
        for c in self.pool.layers:
            for i in range(len(PROMPTS)):
                k, v = (torch.randn((PROMPTS[i], HKV, D), generator=gen, device=cuda).to(BF16) for _ in range(2))
                t = b.tables([i])[0][0].astype(np.int64)
                pos = np.arange(PROMPTS[i])
                c.append(k, v, torch.from_numpy(t[pos // BS] * BS + pos % BS).to(cuda))
        self.state = self.pool.lend(self.ids, 40)
        new = lambda *shape, dt=BF16: torch.zeros(shape, dtype=dt, device=cuda)  # noqa: E731
        self.q, self.out = ([new(T, HQ, D) for _ in range(LAYERS)] for _ in range(2))
        self.k, self.v = ([new(T, HKV, D) for _ in range(LAYERS)] for _ in range(2))
        self.new_lens, self.parents = new(5, dt=torch.int32), new(T, dt=torch.int32)
        self.draft, self.target = new(T, dt=torch.int64), new(T, dt=torch.int64)
        self.freq, self.rscale = rotary_frequencies(48, 1e4, scaling=dict(rope_type="linear", factor=2.0), device=cuda)
        self.step = TreeStep(self.pool.layers, self.q, self.k, self.v, self.out, self.state, self.new_lens, self.parents,
                             self.draft, self.target, D ** -0.5, NODES, 900, DEPTH, inv_freq=self.freq,
                             rotary_scale=self.rscale, shared_blocks=True)

    def fill(self, i):
        """Step i's inputs: the model's and the sampler's part, made up (tokens of a small vocabulary)."""
        rng = np.random.default_rng(i)
        new = rng.integers(1, 20, 5)
        new[i % 5] = 0 if i % 2 else 1
        p = np.full(T, -1, np.int32)
        at = 0
        for n in new:
            p[at + 1:at + n] = [rng.integers(max(0, j - 3), j) for j in range(1, n)]
            at += n
        for dst, x in ((self.new_lens, new), (self.parents, p), (self.draft, rng.integers(0, 3, T)),
                       (self.target, rng.integers(0, 3, T))):
            dst.copy_(torch.from_numpy(np.asarray(x)))
        gen = torch.Generator(device=self.q[0].device).manual_seed(i)
        for x in (*self.q, *self.k, *self.v):
            x.normal_(generator=gen)

    def host(self):
        return [x.cpu().numpy().copy() for x in (self.state.block_table, self.state.held_blocks, self.state.seq_lens,
                                                 self.new_lens, self.state.free_blocks, self.state.taken, self.parents,
                                                 self.draft, self.target)]

    def caches(self):
        out = []
        for c in self.pool.layers:
            scales = (None, None) if c.kv_dtype == "bf16" else (c.k_scale.cpu().numpy().copy(), c.v_scale.cpu().numpy().copy())
            out.append((bits_of(c.k).copy(), bits_of(c.v).copy(), *scales))
        return out


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
def test_steps_against_the_oracle(cuda, kv):
    p = Program(cuda, kv)
    accepted_all = 0
    for i in range(6):
        p.fill(i)
        bt, held, lens, new, free, taken, parents, draft, target = p.host()
        before = p.caches()
        raw = [(paged.bf16_to_f32(bits_of(q)), paged.bf16_to_f32(bits_of(k))) for q, k in zip(p.q, p.k)]
        p.step.begin()
        want = tree.extend_tables(bt, held, lens, new, free, int(taken[0]), BS, T, parents=parents, max_nodes=NODES)
        m = p.step.maps
        np.testing.assert_array_equal(p.state.block_table.cpu(), want["block_table"])
        for name in ("context_lens", "cu_seqlens_q", "slot_mapping", "positions", "tree_mask", "held_blocks"):
            np.testing.assert_array_equal(getattr(m, name).cpu(), want[name], err_msg=name)
        assert int(m.refused) == want["refused"] == 0 and int(p.state.taken) == want["taken"]
        p.step.run()
        rows = int(new.sum())
        for layer, (k, v, ks, vs) in enumerate(before):
            for got, x in zip((p.q[layer], p.k[layer]), raw[layer]):
                turned = tree.rotary(x, want["positions"], p.freq.cpu().numpy(), scale=p.rscale)
                length = np.hypot(x[..., :24], x[..., 24:48])
                err = np.abs(paged.bf16_to_f32(bits_of(got)) - turned)[:rows]
                bound = np.concatenate([length, length, np.zeros_like(x[..., 48:])], -1)[:rows] * 2.0**-8
                assert (err <= bound + 1e-6).all()
            rk, rv = bits_of(p.k[layer]), bits_of(p.v[layer])
            if ks is None:
                paged.append_bf16(k, v, rk, rv, want["slot_mapping"])
                vals = [paged.bf16_to_f32(x) for x in paged.logical_kv(k, v)]
            else:
                paged.append_fp8(k, v, ks, vs, rk, rv, want["slot_mapping"])
                kl = np.ascontiguousarray(paged.k_logical(k)).reshape(len(k), BS, HKV, D)
                vals = [fp8.dequantize(x, s[:, None, :, None]) for x, s in ((kl, ks), (paged.v_logical(v), vs))]
            ref = tree.tree_gqa(paged.bf16_to_f32(bits_of(p.q[layer])), *vals, block_table=want["block_table"],
                                seq_lens=want["context_lens"], cu_seqlens_q=want["cu_seqlens_q"],
                                tree_mask=want["tree_mask"], scale=D ** -0.5)
            check_attention(paged.bf16_to_f32(bits_of(p.out[layer]))[:rows], ref[:rows], f"step {i} layer {layer}")
        p.step.finish()
        acc, path, nxt, after = tree.accept_tree(draft, parents, target, want["cu_seqlens_q"], lens, want["context_lens"], DEPTH)
        a = p.step.accepted
        for got, w in zip(a, (acc, path, nxt, after)):
            np.testing.assert_array_equal(got.cpu(), w)
        np.testing.assert_array_equal(p.state.seq_lens.cpu(), after)
        accepted_all += int(acc.sum())
        for (k, v, ks, vs), now in zip(before, p.caches()):
            tree.compact(k, v, ks, vs, want["block_table"], lens, path, acc)
            for x, y in zip((k, v, ks, vs), now):
                assert x is None or np.array_equal(x, y)
    assert accepted_all > 30  # (paths of several nodes were moved)
    lens = p.state.seq_lens.tolist()
    p.pool.settle(p.state)
    assert [p.pool.blocks.seq_len(s) for s in p.ids] == lens
    p.pool.append_slots(p.ids)


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
def test_captured_steps_are_the_eager_ones(cuda, kv):
    """The three calls captured, replayed with new inputs over carried state; the eager program between them."""
    eager, graphed = Program(cuda, kv), Program(cuda, kv)
    stream = torch.cuda.Stream(cuda)
    graph = torch.cuda.CUDAGraph()
    graphed.fill(0)
    graphed.new_lens.zero_()  # a first step of nothing leaves the state as it is
    for call in (graphed.step.begin, graphed.step.run, graphed.step.finish):
        call()
    assert torch.equal(graphed.state.seq_lens, eager.state.seq_lens)
    stream.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.graph(graph, stream=stream):
        graphed.step.begin()
        graphed.step.run()
        graphed.step.finish()
    torch.cuda.current_stream(cuda).wait_stream(stream)
    for i in range(5):
        for p in (eager, graphed):
            p.fill(i)
        graph.replay()
        eager.step.begin()
        eager.step.run()
        eager.step.finish()
        torch.cuda.synchronize()
        rows = int(eager.new_lens.sum())
        for x, y in zip(eager.out, graphed.out):
            assert torch.equal(x[:rows], y[:rows]), i
        for x, y in zip((*eager.step.accepted, eager.state.seq_lens, eager.state.block_table, eager.state.taken),
                        (*graphed.step.accepted, graphed.state.seq_lens, graphed.state.block_table, graphed.state.taken)):
            assert torch.equal(x, y), i
        for x, y in zip(eager.caches(), graphed.caches()):
            for u, w in zip(x, y):
                assert u is None or np.array_equal(u, w), i


def test_refusals_and_sleep(cuda):
    p = Program(cuda, "bf16")
    ok = dict(caches=p.pool.layers, q=p.q, key=p.k, value=p.v, out=p.out, state=p.state, new_lens=p.new_lens,
              parents=p.parents, draft_tokens=p.draft, target_tokens=p.target, scale=1.0, max_nodes=64, max_seq_len=900,
              max_depth=8, inv_freq=p.freq)
    TreeStep(**ok)
    for bad in (dict(caches=[]), dict(q=p.q[:1]), dict(max_nodes=0), dict(max_nodes=65), dict(max_nodes=320),
                dict(max_depth=0), dict(max_depth=65), dict(new_lens=p.new_lens[:4]), dict(parents=p.parents.long()),
                dict(target_tokens=p.target[:-1]), dict(inv_freq=p.freq.float()), dict(q=[x.float() for x in p.q]),
                dict(value=[x[:, :1] for x in p.v]), dict(inv_freq=torch.zeros(33, dtype=torch.float64, device=cuda))):
        with pytest.raises(ValueError):
            TreeStep(**{**ok, **bad})
    p.pool.settle(p.state)
    for s in p.ids:
        p.pool.blocks.free(s)
    p.pool.sleep()
    with pytest.raises(RuntimeError, match="asleep"):
        p.step.step_layer(0)
    with pytest.raises(RuntimeError, match="asleep"):
        p.step.finish()
