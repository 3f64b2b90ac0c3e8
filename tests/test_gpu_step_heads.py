"""Plans that norm and turn their heads on the way to the cache, against the same plans over heads that norm_rotary (apply_rotary)
has normed and turned before: caches bit for bit. The attention of a decode step then reads its new token from the cache in
the place of the projections: the same values, but probabilities against another reference. Each result rounds
its probabilities to bf16, by 2^-9 of each at most, so two are apart by at most 2 x 2^-9 sum(p |v|) <= 2^-8 max |v| before
their own rounding, 2^-9 of each (values here are below 5). Prompts and trees read it from the cache either way."""

import numpy as np
import pytest
import torch
from kvcase import bits_of

from wavelet_amd import (KVPool, MLALatentCache, PagedKVCache, mla_rotary_append, norm_rotary, rotary_append, rotary_axes,
                         rotary_frequencies)
from wavelet_amd.plan import DecodeStep, GraphDecodeStep, Heads, MLADecodeStep, PrefillStep, TreeStep

pytestmark = pytest.mark.gpu

HQ, HKV, D, BS, LAYERS = 8, 2, 64, 16, 2


def _held(c):
    return [bits_of(c.k), bits_of(c.v)] + ([] if c.k_scale is None else [c.k_scale.cpu().numpy(), c.v_scale.cpu().numpy()])


def _same(a, b):
    for x, y in zip(_held(a), _held(b)):
        np.testing.assert_array_equal(x, y)


class Two:
    """The same inputs twice, and the heads' norm and rotation."""

    def __init__(self, cuda, kv, tokens, seed, axes=False):
        self.g = torch.Generator(device=cuda).manual_seed(seed)
        self.pairs = [[PagedKVCache(24, BS, HKV, D, kv_dtype=kv, device=cuda) for _ in range(LAYERS)] for _ in range(2)]
        z = lambda h: [torch.zeros((tokens, h, D), dtype=torch.bfloat16, device=cuda) for _ in range(LAYERS)]  # noqa: E731
        self.q, self.k, self.v, self.out = zip(*((z(HQ), z(HKV), z(HKV), z(HQ)) for _ in range(2)))
        self.freq = rotary_frequencies(D, 1e4, device=cuda)[0]
        self.qw, self.kw = ([1 + 0.2 * torch.randn(D, generator=self.g, device=cuda).bfloat16() for _ in range(LAYERS)]
                            for _ in range(2))
        self.pos = torch.zeros((3, tokens) if axes else tokens, dtype=torch.int64, device=cuda)
        self.axes = rotary_axes((12, 10, 10), device=cuda) if axes else None
        self.heads = Heads(self.pos, self.freq, self.axes, q_weight=self.qw, k_weight=self.kw, eps=1e-6)

    def fill(self):
        """New projections; the second's normed and turned."""
        for layer in range(LAYERS):
            for x in (self.q, self.k, self.v):
                x[0][layer].normal_(generator=self.g)
                x[1][layer].copy_(x[0][layer])
            norm_rotary(self.q[1][layer], self.k[1][layer], self.pos, self.freq, q_weight=self.qw[layer],
                        k_weight=self.kw[layer], axes=self.axes, out=(self.q[1][layer], self.k[1][layer]))


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("axes", [False, True])
def test_prompt_then_decode(cuda, kv, axes):
    lens = [37, 5, 20]
    t = Two(cuda, kv, sum(lens), 3, axes)
    table = torch.randperm(24, generator=t.g, device=cuda).int().view(3, 8)
    seq = torch.repeat_interleave(torch.arange(3, device=cuda), torch.tensor(lens, device=cuda))
    pos = torch.cat([torch.arange(n, device=cuda) for n in lens])
    t.pos.copy_(pos if not axes else torch.stack([pos, pos // 2, pos % 5]))
    slots = table[seq, pos // BS].long() * BS + pos % BS
    seq_lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, 37, 42, 62], dtype=torch.int32, device=cuda)
    t.fill()
    keys = [x.clone() for x in t.k[0]]
    for i in range(2):
        PrefillStep(t.pairs[i], t.q[i], t.k[i], t.v[i], t.out[i], table, seq_lens, cu, slots, D ** -0.5, 37, 128,
                    heads=t.heads if i == 0 else None).run()
    for layer in range(LAYERS):
        _same(t.pairs[0][layer], t.pairs[1][layer])
        assert torch.equal(t.out[0][layer], t.out[1][layer]) and torch.equal(t.k[0][layer], keys[layer])
        assert torch.equal(t.q[0][layer], t.q[1][layer])
    caches = t.pairs
    t = Two(cuda, kv, 3, 4, axes)
    slots = torch.zeros(3, dtype=torch.int64, device=cuda)
    steps = [DecodeStep(caches[i], t.q[i], t.k[i], t.v[i], t.out[i], table, seq_lens, slots, D ** -0.5, 128,
                        heads=t.heads if i == 0 else None) for i in range(2)]
    for _ in range(20):
        p = seq_lens.long()
        seq_lens += 1
        t.pos.copy_(p if not axes else torch.stack([p, p // 2, p % 5]))
        slots.copy_(table[torch.arange(3, device=cuda), p // BS].long() * BS + p % BS)
        t.fill()
        for s in steps:
            s.run()
        for layer in range(LAYERS):
            _same(caches[0][layer], caches[1][layer])
            torch.testing.assert_close(t.out[0][layer].float(), t.out[1][layer].float(), rtol=2.0 ** -7, atol=5 * 2.0 ** -8)
    if axes:
        return
    graph = GraphDecodeStep(steps[0])  # (heads in place, then the fused append)
    for _ in range(3):
        p = seq_lens.long()
        seq_lens += 1
        t.pos.copy_(p)
        slots.copy_(table[torch.arange(3, device=cuda), p // BS].long() * BS + p % BS)
        t.fill()
        graph.replay()
        steps[1].run()
        for layer in range(LAYERS):
            _same(caches[0][layer], caches[1][layer])
            assert torch.equal(t.out[0][layer], t.out[1][layer])


def _decode_pair(cuda, kv, batch, make_heads, seed, per=2, start=0, **plan):
    """Two decode plans over inputs that are the same (``per`` blocks a sequence, ``start`` tokens in each): their parts,
    and a function that refills both."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    caches = [[PagedKVCache(per * batch, BS, HKV, D, kv_dtype=kv, device=cuda) for _ in range(LAYERS)] for _ in range(2)]
    for a, b in zip(*caches):
        x, y = (torch.randn((per * batch * BS, HKV, D), generator=g, device=cuda).bfloat16() for _ in range(2))
        for c in (a, b):
            c.append(x, y, torch.arange(per * batch * BS, device=cuda))
    z = lambda h: [torch.zeros((batch, h, D), dtype=torch.bfloat16, device=cuda) for _ in range(LAYERS)]  # noqa: E731
    bufs = [(z(HQ), z(HKV), z(HKV), z(HQ)) for _ in range(2)]
    table = torch.randperm(per * batch, generator=g, device=cuda).int().view(batch, per)
    lens, slots = (torch.full((batch,), n, dtype=dt, device=cuda) for n, dt in ((start, torch.int32), (0, torch.int64)))
    pos3 = torch.zeros((3, batch), dtype=torch.int64, device=cuda)
    steps = [DecodeStep(caches[i], *bufs[i], table, lens, slots, D ** -0.5, per * BS, heads=make_heads(i, pos3), **plan)
             for i in range(2)]

    def fill():
        p = lens.long()
        lens.add_(1)
        slots.copy_(table[torch.arange(batch, device=cuda), p // BS].long() * BS + p % BS)
        pos3.copy_(torch.randint(0, 1 << 17, pos3.shape, generator=g, device=cuda))
        for layer in range(LAYERS):
            for x, y in zip(bufs[0][:3], bufs[1][:3]):
                x[layer].normal_(generator=g)
                y[layer].copy_(x[layer])

    return caches, bufs, steps, fill


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("axes", [False, True])
@pytest.mark.parametrize("batch,per,start,part", [(256, 2, 0, 0), (3, 64, 1000, 128)])
def test_turned_alone_and_captured(cuda, kv, axes, batch, per, start, part):
    """Heads with a rotation and no norm: a captured plan leaves the queries and the cache that the same plan leaves when it
    is run, also where a context is shared out and merged; its attention takes the new token from its buffers."""
    freq = rotary_frequencies(D, 1e4, device=cuda)[0]
    of = rotary_axes((12, 10, 10), device=cuda) if axes else None
    caches, bufs, steps, fill = _decode_pair(
        cuda, kv, batch, lambda i, pos: Heads(pos if axes else pos[0], freq, of, scale=1.25), 21, per, start,
        partition_size=part)
    graph = GraphDecodeStep(steps[1])
    for _ in range(5):
        fill()
        keys = [x.clone() for x in bufs[0][1]]
        steps[0].run()
        graph.replay()
        for layer in range(LAYERS):
            assert torch.equal(bufs[0][0][layer], bufs[1][0][layer]) and torch.equal(bufs[0][1][layer], keys[layer])
            _same(caches[0][layer], caches[1][layer])
            torch.testing.assert_close(bufs[0][3][layer].float(), bufs[1][3][layer].float(), rtol=2.0 ** -7, atol=5 * 2.0 ** -8)


KINDS = {  # what a plan's heads may be: (turned, several axes, normed, weights, offset)
    "turned": (True, False, False, False, 0.0), "turned by axes": (True, True, False, False, 0.0),
    "normed": (False, False, True, True, 0.0), "normed without weights": (False, False, True, False, 0.0),
    "both, without weights": (True, False, True, False, 0.0), "both by axes": (True, True, True, True, 1.0),
}


class Kind:
    """Heads of a kind, and the same by ``rotary_append`` alone."""

    def __init__(self, cuda, kind, pos3, seed=0):
        turned, axes, normed, weights, offset = KINDS[kind]
        g = torch.Generator(device=cuda).manual_seed(seed)
        how = {}
        if turned:
            how.update(positions=pos3 if axes else pos3[0], inv_freq=rotary_frequencies(48, 1e4, device=cuda)[0], scale=1.25,
                       interleaved=True, axes=rotary_axes((10, 8, 6), device=cuda) if axes else None)
        if normed:
            how.update(eps=1e-5, weight_offset=offset)
        self.how = how
        self.w = [[1 + 0.2 * torch.randn(D, generator=g, device=cuda) for _ in range(LAYERS)] for _ in range(2)] if weights else None
        self.heads = Heads(**how) if not weights else Heads(q_weight=self.w[0], k_weight=self.w[1], **how)

    def append(self, layer, q, key, value, cache, slots):
        w = {} if self.w is None else dict(q_weight=self.w[0][layer], k_weight=self.w[1][layer])
        rotary_append(q, key, value, cache, slots, out=q, **w, **self.how)


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("groups", [False, True])
def test_kinds_of_heads_in_a_decode_step(cuda, kind, kv, groups):
    """A plan, and but for groups a captured one, against rotary_append and the plan's attention alone; a captured plan's
    attention takes the new token from its buffers (the tolerance above)."""
    batch, made = 6, {}

    def make(i, pos):
        made["of"] = Kind(cuda, kind, pos)
        return made["of"].heads if i == 0 else None

    more = dict(group_size=3, prefix_lens=torch.tensor([32, 16], dtype=torch.int32, device=cuda), max_prefix_len=32) if groups else {}
    caches, bufs, steps, fill = _decode_pair(cuda, kv, batch, make, 31, 8, 60, **more)
    runs = [steps[0].run] if groups else [steps[0].run, GraphDecodeStep(steps[0]).replay]
    for n in range(6):
        fill()
        keys = [x.clone() for x in bufs[0][1]]
        captured = n % len(runs) == 1
        runs[n % len(runs)]()
        steps[1].prepare()
        for layer in range(LAYERS):
            q, k, v, out = (x[layer] for x in bufs[1])
            made["of"].append(layer, q, k, v, caches[1][layer], steps[1].slot_mapping)
            steps[1].attend(layer)
            assert torch.equal(bufs[0][0][layer], q)
            _same(caches[0][layer], caches[1][layer])
            if captured:
                torch.testing.assert_close(bufs[0][3][layer].float(), out.float(), rtol=2.0 ** -7, atol=5 * 2.0 ** -8)
            else:
                assert torch.equal(bufs[0][3][layer], out) and torch.equal(bufs[0][1][layer], keys[layer])


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("kind", KINDS)
def test_kinds_of_heads_in_a_prompt(cuda, kind, kv):
    lens = [37, 5, 20]
    g = torch.Generator(device=cuda).manual_seed(41)
    pairs = [[PagedKVCache(24, BS, HKV, D, kv_dtype=kv, device=cuda) for _ in range(LAYERS)] for _ in range(2)]
    bufs = [[torch.randn((62, h, D), generator=g, device=cuda).bfloat16() for _ in range(LAYERS)] for h in (HQ, HKV, HKV, HQ)]
    bufs = [[[x.clone() for x in of] for of in bufs] for _ in range(2)]
    table = torch.randperm(24, generator=g, device=cuda).int().view(3, 8)
    seq = torch.repeat_interleave(torch.arange(3, device=cuda), torch.tensor(lens, device=cuda))
    pos = torch.cat([torch.arange(n, device=cuda) for n in lens])
    slots = table[seq, pos // BS].long() * BS + pos % BS
    seq_lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, 37, 42, 62], dtype=torch.int32, device=cuda)
    of = Kind(cuda, kind, torch.stack([pos + 70000, pos // 2, pos % 5]))
    steps = [PrefillStep(pairs[i], *bufs[i], table, seq_lens, cu, slots, D ** -0.5, 37, 128, heads=of.heads if i == 0 else None)
             for i in range(2)]
    steps[0].run()
    for layer in range(LAYERS):
        q, k, v, out = (x[layer] for x in bufs[1])
        of.append(layer, q, k, v, pairs[1][layer], slots)
        steps[1].attend(layer)
        _same(pairs[0][layer], pairs[1][layer])
        for a, b in zip(bufs[0], (q, k, v, out)):
            assert torch.equal(a[layer], b)


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("kind", [k for k in KINDS if "axes" not in k])
def test_kinds_of_heads_in_a_drafted_step(cuda, kind, kv):
    """Against the same step over heads that rotary_append has normed and turned into a cache of their own."""
    rows, g = 24, torch.Generator(device=cuda).manual_seed(51)
    x = [[torch.randn((rows, h, D), generator=g, device=cuda).bfloat16() for _ in range(LAYERS)] for h in (HQ, HKV, HKV, HQ)]
    new = torch.tensor([9, 1], dtype=torch.int32, device=cuda)
    parents = torch.full((rows,), -1, dtype=torch.int32, device=cuda)
    parents[1:9] = torch.tensor([0, 0, 1, 2, 3, 3, 4, 0], device=cuda)
    draft, target = (torch.randint(0, 2, (rows,), generator=g, device=cuda) for _ in range(2))
    got = []
    for i in range(2):
        bufs = [[t.clone() for t in of] for of in x]
        pool = KVPool(LAYERS, 24, BS, HKV, D, kv, device=cuda, max_model_len=96)
        for j, n in enumerate((30, 4)):
            pool.blocks.allocate(j, np.arange(n) + 1000 * j)
        state = pool.lend([0, 1], 12)
        kw = {}
        if i == 0:
            of = Kind(cuda, kind, torch.zeros((3, rows), dtype=torch.int64, device=cuda))
            of.heads.positions = None  # (they are the step's)
            kw["heads"] = of.heads
        step = TreeStep(pool.layers, *bufs, state, new, parents, draft, target, D ** -0.5, 64, 96, 8, **kw)
        step.begin()
        if i == 1:
            at = torch.arange(rows, device=cuda)
            of = Kind(cuda, kind, torch.stack([step.maps.positions] * 3))
            for layer in range(LAYERS):
                c = PagedKVCache(-(-rows // BS), BS, HKV, D, device=cuda)
                of.append(layer, bufs[0][layer], bufs[1][layer], bufs[2][layer], c, at)
                bufs[1][layer].copy_(c.k.permute(0, 3, 1, 2, 4).reshape(-1, HKV, D)[:rows])
        step.run()
        step.finish()
        got.append((pool, state, bufs, step))
    a, b = got
    for layer in range(LAYERS):
        _same(a[0].layers[layer], b[0].layers[layer])
        assert torch.equal(a[2][3][layer][:10], b[2][3][layer][:10]) and torch.equal(a[2][0][layer][:10], b[2][0][layer][:10])
        assert torch.equal(a[2][1][layer], x[1][layer])
    assert torch.equal(a[1].seq_lens, b[1].seq_lens) and torch.equal(a[3].accepted.path, b[3].accepted.path)


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
def test_drafted_steps(cuda, kv):
    rows = 48
    prompts = (40, 3, 16)
    programs = []
    for i in range(2):
        t = Two(cuda, kv, rows, 7)
        pool = KVPool(LAYERS, 24, BS, HKV, D, kv, device=cuda, max_model_len=128)
        for j, n in enumerate(prompts):
            pool.blocks.allocate(j, np.arange(n) + 1000 * j)
        state = pool.lend([0, 1, 2], 12)
        new, parents = (torch.zeros(n, dtype=torch.int32, device=cuda) for n in (3, rows))
        draft, target = (torch.zeros(rows, dtype=torch.int64, device=cuda) for _ in range(2))
        heads = Heads(inv_freq=t.freq, q_weight=t.qw, k_weight=t.kw, eps=1e-6) if i == 0 else None
        step = TreeStep(pool.layers, t.q[0], t.k[0], t.v[0], t.out[0], state, new, parents, draft, target, D ** -0.5, 64, 128,
                        8, heads=heads)
        programs.append((t, pool, state, new, parents, draft, target, step))
    for n in range(4):
        rng = np.random.default_rng(n)
        lens = rng.integers(1, 12, 3)
        p = np.full(rows, -1, np.int32)
        at = 0
        for m in lens:
            p[at + 1:at + m] = [rng.integers(max(0, j - 3), j) for j in range(1, m)]
            at += m
        toks = rng.integers(0, 3, (2, rows))
        for i, (t, pool, state, new, parents, draft, target, step) in enumerate(programs):
            for dst, x in ((new, lens), (parents, p), (draft, toks[0]), (target, toks[1])):
                dst.copy_(torch.from_numpy(np.asarray(x)))
            t.g.manual_seed(n)
            for x in (*t.q[0], *t.k[0], *t.v[0]):
                x.normal_(generator=t.g)
            step.begin()
            if i == 1:  # (rows past the step's last have no position)
                for layer in range(LAYERS):
                    norm_rotary(t.q[0][layer], t.k[0][layer], step.maps.positions, t.freq, q_weight=t.qw[layer],
                                k_weight=t.kw[layer], out=(t.q[0][layer], t.k[0][layer]))
            step.run()
            step.finish()
        a, b = programs
        for layer in range(LAYERS):
            _same(a[1].layers[layer], b[1].layers[layer])
            assert torch.equal(a[0].out[0][layer][:at], b[0].out[0][layer][:at])
        assert torch.equal(a[2].seq_lens, b[2].seq_lens) and torch.equal(a[7].accepted.path, b[7].accepted.path)


def test_latent_decode(cuda):
    g = torch.Generator(device=cuda).manual_seed(11)
    heads_n, batch = 16, 3
    pairs = [[MLALatentCache(12, BS, device=cuda) for _ in range(LAYERS)] for _ in range(2)]
    z = lambda *s: [torch.zeros(s, dtype=torch.bfloat16, device=cuda) for _ in range(LAYERS)]  # noqa: E731
    bufs = [(z(batch, heads_n, 512), z(batch, heads_n, 64), z(batch, 512), z(batch, 64), z(batch, heads_n, 512)) for _ in range(2)]
    freq = rotary_frequencies(64, 1e4, device=cuda)[0]
    pos, slots = (torch.zeros(batch, dtype=torch.int64, device=cuda) for _ in range(2))
    weights = [1 + 0.2 * torch.randn(512, generator=g, device=cuda).bfloat16() for _ in range(LAYERS)]
    table = torch.randperm(12, generator=g, device=cuda).int().view(3, 4)
    lens = torch.zeros(batch, dtype=torch.int32, device=cuda)
    steps = [MLADecodeStep(pairs[i], *bufs[i], table, lens, slots, 0.05, 64,
                           heads=Heads(pos, freq, interleaved=True, k_weight=weights, eps=1e-6) if i == 0 else None)
             for i in range(2)]
    for _ in range(18):
        pos.copy_(lens)
        lens += 1
        slots.copy_(table[torch.arange(3, device=cuda), pos // BS].long() * BS + pos % BS)
        for layer in range(LAYERS):
            for j in range(4):
                bufs[0][j][layer].normal_(generator=g)
                bufs[1][j][layer].copy_(bufs[0][j][layer])
            qp, kc, kp = bufs[1][1][layer], bufs[1][2][layer], bufs[1][3][layer]
            # (turned without a norm: apply_rotary's angles are rounded otherwise)
            alone = MLALatentCache(1, BS, device=cuda)
            mla_rotary_append(qp, kc, kp, alone, torch.arange(3, device=cuda), pos, freq, interleaved=True, out=qp)
            kp.copy_(alone.latent[0, :3, 512:])
            norm_rotary(kc[:, None], None, q_weight=weights[layer], eps=1e-6, out=(kc[:, None], None))
        for s in steps:
            s.run()
        for layer in range(LAYERS):
            a, b = (p[layer].latent for p in pairs)
            # (the entry's squares are added in another order than norm_rotary adds them: at most a rounding apart)
            torch.testing.assert_close(a.float(), b.float(), rtol=2.0 ** -7, atol=0)
            assert torch.equal(a[..., 512:], b[..., 512:]) and torch.equal(bufs[0][1][layer], bufs[1][1][layer])
            b.copy_(a)  # over one cache the attentions agree bit for bit
            steps[1].attend(layer)
            assert torch.equal(bufs[0][4][layer], bufs[1][4][layer])


def test_plans_keep_what_they_were_built_with(cuda):
    """Fields of the heads that are set anew, and lists changed, after the plan was built."""
    t = Two(cuda, "bf16", 2, 5)
    table = torch.arange(4, dtype=torch.int32, device=cuda).view(2, 2)
    lens, slots = torch.tensor([1, 1], dtype=torch.int32, device=cuda), torch.tensor([0, 32], device=cuda)
    heads = Heads(t.pos, t.freq, q_weight=list(t.qw), k_weight=list(t.kw), eps=1e-6)
    step = DecodeStep(t.pairs[0], t.q[0], t.k[0], t.v[0], t.out[0], table, lens, slots, D ** -0.5, 32, heads=heads)
    heads.positions = heads.inv_freq = None
    heads.q_weight[:] = heads.k_weight[:] = [None] * LAYERS
    assert step.heads.positions is t.pos and step.heads.inv_freq is t.freq
    assert all(a is b for a, b in zip(step.heads.q_weight + step.heads.k_weight, t.qw + t.kw))
    other = DecodeStep(t.pairs[1], t.q[1], t.k[1], t.v[1], t.out[1], table, lens, slots, D ** -0.5, 32)
    t.pos.copy_(torch.tensor([0, 7], device=cuda))
    for run in (step.run, GraphDecodeStep(step).replay):
        t.fill()
        run()
        other.run()
        for layer in range(LAYERS):
            _same(t.pairs[0][layer], t.pairs[1][layer])


def test_refusals(cuda):
    t = Two(cuda, "bf16", 2, 1)
    table, lens = torch.zeros((2, 2), dtype=torch.int32, device=cuda), torch.ones(2, dtype=torch.int32, device=cuda)
    slots = torch.zeros(2, dtype=torch.int64, device=cuda)
    args = (t.pairs[0], t.q[0], t.k[0], t.v[0], t.out[0], table, lens, slots, 0.125, 32)
    DecodeStep(*args, heads=t.heads)
    for bad in (Heads(), Heads(t.pos), Heads(None, t.freq), Heads(t.pos[:1], t.freq), Heads(t.pos, t.freq, q_weight=t.qw),
                Heads(t.pos, t.freq, q_weight=t.qw[:1], eps=1e-6), Heads(t.pos, t.freq, k_weight=[w[:8] for w in t.kw], eps=1e-6),
                Heads(torch.zeros(4, dtype=torch.int64, device=cuda)[::2], t.freq), Heads(eps=1e-6, axes=t.pos.int())):
        with pytest.raises(ValueError):
            DecodeStep(*args, heads=bad)
    lat = [MLALatentCache(2, BS, device=cuda)]
    z = lambda *s: [torch.zeros(s, dtype=torch.bfloat16, device=cuda)]  # noqa: E731
    with pytest.raises(ValueError, match="rotation"):
        MLADecodeStep(lat, z(2, 16, 512), z(2, 16, 64), z(2, 512), z(2, 64), z(2, 16, 512), table, lens, slots, 0.1, 32,
                      heads=Heads(eps=1e-6))
