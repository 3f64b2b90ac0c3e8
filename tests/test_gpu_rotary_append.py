"""The append with norm and rotation on the way: the queries and keys against the float64 oracle (bounds:
headcase.py), the cache bit for bit against the oracle's append of the keys that norm_rotary rounds (without a norm: that a
bf16 cache holds, each at a slot of its own)."""

import numpy as np
import pytest
import torch
from headcase import U, check, check_forward, f64, size
from kvcase import assert_guards, bits_of, guard_cache

from oracle import heads, paged
from wavelet_amd import (MLALatentCache, PagedKVCache, mla_rotary_append, norm_rotary, paged_decode_gqa,
                         prefill_gqa, rotary_append, rotary_axes, rotary_frequencies)

pytestmark = pytest.mark.gpu


def _slots(rng, lens, ctx, block, spare=3):
    """Slots of new tokens of sequences whose blocks are dealt from a shuffled pool, and the number of blocks."""
    need = [-(-(c + n) // block) for c, n in zip(ctx, lens)]
    perm = rng.permutation(sum(need) + spare)
    out, at = [], 0
    for c, n, m in zip(ctx, lens, need):
        pos = np.arange(c, c + n)
        out.append(perm[at:at + m][pos // block] * block + pos % block)
        at += m
    return np.concatenate(out).astype(np.int64), sum(need) + spare


def _cache(cuda, blocks, block, hk, d, kv, seed=0):
    """A cache that holds something everywhere."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    c = PagedKVCache(blocks, block, hk, d, kv_dtype=kv, device=cuda)
    for t in (c.k, c.v):
        x = torch.randn(t.shape, generator=g, device=cuda)
        t.copy_(x if kv == "bf16" else (x * 100).to(torch.float8_e4m3fn).view(torch.uint8))
    if kv != "bf16":
        for s in (c.k_scale, c.v_scale):
            s.copy_(torch.ldexp(torch.ones_like(s), torch.randint(-9, -3, s.shape, generator=g, device=cuda)))
    return c


def _inputs(cuda, tokens, hq, hk, d, r, weights, seed=1):
    g = torch.Generator(device=cuda).manual_seed(seed + tokens)
    x = torch.randn((tokens, hq + 2 * hk, d), generator=g, device=cuda).bfloat16()
    x *= torch.exp(torch.randn((1, hq + 2 * hk, 1), generator=g, device=cuda)).bfloat16()
    each = weights == "each"
    w = [torch.randn((h, d) if each else (d,), generator=g, device=cuda).to(torch.float32 if each else torch.bfloat16)
         for h in (hq, hk)] if weights else [None, None]
    pos = torch.randint(0, 40000, (tokens,), generator=g, device=cuda)
    return x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], w, pos, rotary_frequencies(r, 1e4, device=cuda)[0] if r else None


def _expected(c, key, value, slots):
    """The oracle's append of bf16 keys and values to a copy of the cache (which knows only slots that are there)."""
    slots = np.where(slots < c.num_blocks * c.block_size, slots, -1)
    arrays = [bits_of(t).copy() for t in (c.k, c.v)]
    if c.kv_dtype == "bf16":
        paged.append_bf16(*arrays, bits_of(key), bits_of(value), slots)
        return arrays
    scales = [t.cpu().numpy().copy() for t in (c.k_scale, c.v_scale)]
    paged.append_fp8(*arrays, *scales, bits_of(key), bits_of(value), slots)
    return arrays + scales


def _held(c):
    return [bits_of(t) for t in (c.k, c.v)] + ([] if c.k_scale is None else [t.cpu().numpy() for t in (c.k_scale, c.v_scale)])


def _run(cuda, q, key, value, c, slots, w, pos, freq, eps, **how):
    guards = guard_cache(c)
    norm = {} if eps is None else dict(q_weight=w[0], k_weight=w[1], eps=eps)
    if eps is None:
        want_q, want_k = _turned(cuda, q, key, value, pos, freq, how)
    else:
        want_q, want_k = norm_rotary(q, key, pos, freq, **norm, **how)
    want = _expected(c, want_k, value, slots)
    before = [t.clone() for t in (q, key, value)]
    got = rotary_append(q, key, value, c, torch.from_numpy(slots).to(cuda), pos, freq, **norm, **how)
    assert_guards(guards, "rotary_append")
    assert torch.equal(got, want_q)
    for a, b in zip(_held(c), want):
        np.testing.assert_array_equal(a, b)
    for a, b in zip((q, key, value), before):
        assert torch.equal(a, b)
    return got


def _turned(cuda, q, key, value, pos, freq, how):
    """Queries and keys as they are turned without a norm, checked against the oracle."""
    tokens, hk, d = key.shape
    c = PagedKVCache(-(-tokens // 16), 16, hk, d, device=cuda)
    got = rotary_append(q, key, value, c, torch.arange(tokens, device=cuda), pos, freq, **how)
    k = c.k.permute(0, 3, 1, 2, 4).reshape(-1, hk, d)[:tokens].contiguous()
    axes, inter, scale = how.get("axes"), how.get("interleaved", False), how.get("scale", 1.0)
    angle = heads.phases(f64(pos), f64(freq), None if axes is None else axes.cpu().numpy())
    for y, x in ((got, q), (k, key)):
        check(y, heads.turn(f64(x), angle, inter, scale), 16 * U * size(f64(x), angle.shape[1], inter, scale), "turned")
    return got, k


SHAPES = [  # head layout, new tokens, contexts, block size
    ((32, 8, 128), [1] * 9, [0, 1, 15, 16, 17, 31, 40, 100, 255], 16),
    ((14, 2, 64), [5, 1, 33], [3, 16, 0], 16),
    ((28, 4, 128), [37, 90, 16], [0, 7, 60], 64),
    ((16, 5, 64), [70, 300], [130, 0], 128),
    ((4, 4, 128), [600, 513], [5, 250], 256),
    ((8, 1, 64), [700, 411, 300], [9, 0, 16], 32),
    ((3, 3, 64), [4096, 37], [0, 11], 16),
    ((2, 1, 128), [1100], [5], 48),
    ((4, 8, 64), [8192, 9], [0, 5], 16),
]


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_as_the_oracle_appends(cuda, case, kv):
    (hq, hk, d), new, ctx, block = SHAPES[case]
    rng = np.random.default_rng(case)
    slots, blocks = _slots(rng, new, ctx, block)
    for r, inter, eps, weights in ((d, False, 1e-6, "dim"), (d, True, None, None), (d // 2, False, 1e-5, "each"),
                                   (20, False, 1e-6, None), (26, True, 1e-6, "dim")):
        q, key, value, w, pos, freq = _inputs(cuda, len(slots), hq, hk, d, r, weights)
        got = _run(cuda, q, key, value, _cache(cuda, blocks, block, hk, d, kv), slots, w, pos, freq, eps,
                   interleaved=inter, scale=1.25)
        if eps is not None:
            check_forward(got, q, w[0], eps, heads.phases(f64(pos), f64(freq)), 0.0, inter, 1.25)


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("tokens", [40, 1030, 4200])
def test_skipped_slots_and_blocks_that_are_not_there(cuda, tokens, kv):
    """Nothing is written for them; their queries are computed."""
    rng = np.random.default_rng(tokens)
    slots, blocks = _slots(rng, [tokens // 2, tokens - tokens // 2], [3, 18], 16)
    slots[rng.random(tokens) < 0.2] = -1
    slots[rng.random(tokens) < 0.05] = (blocks + 3) * 16
    slots[rng.random(tokens) < 0.05] = -7
    slots[rng.random(tokens) < 0.02] = (1 << 40) + 5
    if kv == "fp8_e4m3":  # a block in one run of a call: what a hole cuts off goes too
        last, seen = None, set()
        for i, s in enumerate(slots):
            b = s // 16 if 0 <= s < blocks * 16 else None
            if b is not None and b != last:
                if b in seen:
                    slots[i] = -1
                    b = None
                else:
                    seen.add(b)
            last = b
    q, key, value, w, pos, freq = _inputs(cuda, tokens, 6, 3, 64, 64, "dim")
    _run(cuda, q, key, value, _cache(cuda, blocks, 16, 3, 64, kv), slots, w, pos, freq, 1e-6)


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
def test_slots_in_another_order(cuda, kv):
    """A block's tokens backwards, and in pairs."""
    rng = np.random.default_rng(3)
    for block, tokens in ((16, 320), (64, 640)):
        slots, blocks = _slots(rng, [tokens], [0], block)
        for i in range(0, tokens, block):
            if i // block % 3 == 0:
                slots[i:i + block] = slots[i:i + block][::-1].copy()
            elif i // block % 3 == 1:
                slots[i:i + block] = slots[i:i + block].reshape(-1, 2)[:, ::-1].reshape(-1).copy()
        q, key, value, w, pos, freq = _inputs(cuda, tokens, 4, 2, 128, 128, "dim")
        _run(cuda, q, key, value, _cache(cuda, blocks, block, 2, 128, kv), slots, w, pos, freq, 1e-6)


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
def test_values_that_are_not_finite(cuda, kv):
    rng = np.random.default_rng(4)
    slots, blocks = _slots(rng, [37, 1, 64], [5, 9, 0], 16)
    q, key, value, w, pos, freq = _inputs(cuda, len(slots), 2, 2, 64, 64, "dim")
    value[3, 0, 5], value[40, 1, 60], value[50, 0, 0] = float("nan"), float("inf"), -float("inf")
    key[11, 1, 7] = float("nan")
    key[37, 0] = 0
    c = _cache(cuda, blocks, 16, 2, 64, kv)
    _, want_k = norm_rotary(q, key, pos, freq, q_weight=w[0], k_weight=w[1])
    want = _expected(c, want_k, value, slots)
    rotary_append(q, key, value, c, torch.from_numpy(slots).to(cuda), pos, freq, q_weight=w[0], k_weight=w[1], eps=1e-6)
    got = _held(c)
    if kv == "bf16":
        for i in range(2):  # (a NaN's bits are its own)
            np.testing.assert_array_equal(paged.bf16_to_f32(got[i]), paged.bf16_to_f32(want[i]))
    else:
        for i in range(2):
            nan = (got[i] & 0x7f) == 0x7f
            np.testing.assert_array_equal(nan, (want[i] & 0x7f) == 0x7f)
            np.testing.assert_array_equal(got[i][~nan], want[i][~nan])
        for i in (2, 3):
            np.testing.assert_array_equal(got[i], want[i])


def test_axes_norm_alone_no_queries_and_in_place(cuda):
    rng = np.random.default_rng(5)
    slots, blocks = _slots(rng, [50, 21], [7, 0], 16)
    q, key, value, w, pos, freq = _inputs(cuda, 71, 4, 2, 128, 128, "dim")
    pos3 = torch.stack([pos, pos // 3, pos // 7])
    axes = rotary_axes((16, 24, 24), device=cuda)
    _run(cuda, q, key, value, _cache(cuda, blocks, 16, 2, 128, "bf16"), slots, w, pos3, freq, 1e-6, axes=axes)
    _run(cuda, q, key, value, _cache(cuda, blocks, 16, 2, 128, "fp8_e4m3"), slots, w, pos3, freq, None, axes=axes)
    _run(cuda, q, key, value, _cache(cuda, blocks, 16, 2, 128, "fp8_e4m3"), slots, w, None, None, 1e-6)
    for kv in ("bf16", "fp8_e4m3"):
        a, b, c = (_cache(cuda, blocks, 16, 2, 128, kv) for _ in range(3))
        at = torch.from_numpy(slots).to(cuda)
        want = rotary_append(q, key, value, a, at, pos, freq, q_weight=w[0], k_weight=w[1], eps=1e-6)
        assert rotary_append(None, key, value, b, at, pos, freq, k_weight=w[1], eps=1e-6) is None
        mine = q.contiguous().clone()
        assert rotary_append(mine, key, value, c, at, pos, freq, q_weight=w[0], k_weight=w[1], eps=1e-6, out=mine) is mine
        assert torch.equal(mine, want)
        for x, y, z in zip(_held(a), _held(b), _held(c)):
            np.testing.assert_array_equal(x, y)
            np.testing.assert_array_equal(x, z)


def _moved(cuda, tensors, shift):
    """The same rows at another alignment."""
    out = [torch.empty(len(t), t.shape[1] * 64 + 9, device=cuda).bfloat16()[:, shift:shift + t.shape[1] * 64].view(t.shape)
           for t in tensors]
    for a, b in zip(out, tensors):
        a.copy_(b)
    return out


@pytest.mark.parametrize("shift", [1, 3])
def test_rows_that_are_not_aligned(cuda, shift):
    rng = np.random.default_rng(6)
    slots, blocks = _slots(rng, [30], [2], 16)
    q, key, value, w, pos, freq = _inputs(cuda, 30, 4, 2, 64, 64, "dim")
    for kv in ("bf16", "fp8_e4m3"):
        _run(cuda, *_moved(cuda, (q, key, value), shift), _cache(cuda, blocks, 16, 2, 64, kv), slots, w, pos, freq, 1e-6)


@pytest.mark.parametrize("shift", [0, 1, 4])
@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
def test_one_row_that_is_not_aligned(cuda, kv, shift):
    """A token whose row of projections is of an odd length, or starts off a 16-byte boundary: contiguous all the same."""
    q, key, value, w, pos, freq = _inputs(cuda, 1, 4, 2, 64, 64, "dim")
    row = torch.zeros((1, shift + 8 * 64 + 3), dtype=torch.bfloat16, device=cuda)
    parts = [row[:, shift + at:shift + at + n].view(1, -1, 64) for at, n in ((0, 256), (256, 128), (384, 128))]
    for p, x in zip(parts, (q, key, value)):
        p.copy_(x)
    slot = torch.tensor([17], device=cuda)
    got, want = (_cache(cuda, 3, 16, 2, 64, kv) for _ in range(2))
    a = rotary_append(parts[0], parts[1], parts[2], got, slot, pos, freq, q_weight=w[0], k_weight=w[1], eps=1e-6)
    b = rotary_append(q.contiguous(), key.contiguous(), value.contiguous(), want, slot, pos, freq, q_weight=w[0],
                      k_weight=w[1], eps=1e-6)
    check_forward(a, q, w[0], 1e-6, heads.phases(f64(pos), f64(freq)), 0.0, False, 1.0)
    check_forward(b, q, w[0], 1e-6, heads.phases(f64(pos), f64(freq)), 0.0, False, 1.0)
    np.testing.assert_array_equal(_held(got)[1], _held(want)[1])
    if kv == "bf16":
        check_forward(got.k[1, :, :, 1].reshape(1, 2, 64), key, w[1], 1e-6, heads.phases(f64(pos), f64(freq)), 0.0, False, 1.0)
    # and appended alone
    alone, packed = (_cache(cuda, 3, 16, 2, 64, kv) for _ in range(2))
    alone.append(parts[1], parts[2], slot)
    packed.append(key.contiguous(), value.contiguous(), slot)
    for x, y in zip(_held(alone), _held(packed)):
        np.testing.assert_array_equal(x, y)


def test_rows_aligned_to_eight_bytes(cuda):
    """norm_rotary takes them two elements at a time, rotary_append one: squares are added in another order."""
    q, key, value, w, pos, freq = _inputs(cuda, 30, 4, 2, 64, 64, "dim")
    c = PagedKVCache(2, 16, 2, 64, device=cuda)
    got = rotary_append(*_moved(cuda, (q, key, value), 4), c, torch.arange(30, device=cuda), pos, freq, q_weight=w[0],
                        k_weight=w[1], eps=1e-6)
    angle = heads.phases(f64(pos), f64(freq))
    check_forward(got, q, w[0], 1e-6, angle, 0.0, False, 1.0)
    check_forward(c.k.permute(0, 3, 1, 2, 4).reshape(-1, 2, 64)[:30], key, w[1], 1e-6, angle, 0.0, False, 1.0)


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("d,r,inter,shift", [(64, 20, False, 0), (128, 20, False, 0), (128, 92, False, 0), (64, 64, True, 4),
                                             (64, 34, False, 0)])
def test_squares_are_added_in_norm_rotary_s_order(cuda, d, r, inter, shift, kv):
    """Pairs that are taken two or one at a time, from values of many sizes, whose sum depends on the order in its last bit
    (and some 1 in 2^16 results with it: tens of these)."""
    rng = np.random.default_rng(r)
    slots, blocks = _slots(rng, [3000, 1096], [0, 5], 16)
    q, key, value, w, pos, freq = _inputs(cuda, len(slots), 16, 8, d, r, "dim")
    g = torch.Generator(device=cuda).manual_seed(1)
    q, key = ((x * torch.exp(2 * torch.randn(x.shape, generator=g, device=cuda))).bfloat16() for x in (q, key))
    if shift:  # (rows aligned to 8 bytes)
        wide = torch.empty((len(slots), 16 * d + 12), device=cuda).bfloat16()[:, shift:shift + 16 * d].view(q.shape)
        q = wide.copy_(q)
    _run(cuda, q, key, value, _cache(cuda, blocks, 16, 8, d, kv), slots, w, pos, freq, 1e-6, interleaved=inter)


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
def test_prompt_and_decode_as_they_are_used(cuda, kv):
    """A prompt and then tokens one by one: rotary_append and the attentions against norm_rotary and theirs. (A decode
    step's two results are apart as test_gpu_step_heads.py derives.)"""
    hq, hk, d, block, new = 8, 2, 128, 16, [37, 5]
    g = torch.Generator(device=cuda).manual_seed(9)
    freq, scale = rotary_frequencies(d, 1e6, device=cuda)
    w = [1 + 0.2 * torch.randn(d, generator=g, device=cuda).bfloat16() for _ in range(2)]
    norm = dict(q_weight=w[0], k_weight=w[1], eps=1e-6)
    a, b = (PagedKVCache(12, block, hk, d, kv_dtype=kv, device=cuda) for _ in range(2))
    table = torch.randperm(12, generator=g, device=cuda).int().view(2, 6)

    def rows(n):
        x = torch.randn((n, hq + 2 * hk, d), generator=g, device=cuda).bfloat16()
        return x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]

    def at(pos, seq):
        return table[seq, pos // block].long() * block + pos % block

    pos = torch.cat([torch.arange(n, device=cuda) for n in new])
    seq = torch.repeat_interleave(torch.arange(2, device=cuda), torch.tensor(new, device=cuda))
    lens = torch.tensor(new, dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, 37, 42], dtype=torch.int32, device=cuda)
    q, key, value = rows(42)
    q1 = rotary_append(q, key, value, a, at(pos, seq), pos, freq, **norm, scale=scale)
    q2, k2 = norm_rotary(q, key, pos, freq, **norm, scale=scale)
    one = prefill_gqa(q1, a, table, lens, cu, d ** -0.5, max_query_len=37, max_seq_len=64)
    two = prefill_gqa(q2, b, table, lens, cu, d ** -0.5, max_query_len=37, max_seq_len=64, key=k2, value=value,
                      slot_mapping=at(pos, seq))
    assert torch.equal(one, two)
    for _ in range(12):
        q, key, value = rows(2)
        pos, lens = lens.long(), lens + 1
        slots = at(pos, torch.arange(2, device=cuda))
        q1 = rotary_append(q, key, value, a, slots, pos, freq, **norm, scale=scale)
        q2, k2 = norm_rotary(q, key, pos, freq, **norm, scale=scale)
        one = paged_decode_gqa(q1, a, table, lens, d ** -0.5, max_seq_len=64)
        two = paged_decode_gqa(q2, b, table, lens, d ** -0.5, max_seq_len=64, new_key=k2, new_value=value,
                               slot_mapping=slots)
        torch.testing.assert_close(one.float(), two.float(), rtol=2.0 ** -7, atol=5 * 2.0 ** -8)
        for x, y in zip(_held(a), _held(b)):
            np.testing.assert_array_equal(x, y)


@pytest.mark.parametrize("rank,rope,heads_n,block,r", [(512, 64, 16, 64, 64), (512, 64, 128, 16, 32), (64, 8, 3, 16, 8),
                                                       (1032, 24, 2, 32, 24), (128, 128, 5, 16, 118)])
@pytest.mark.parametrize("inter", [False, True])
def test_latent(cuda, rank, rope, heads_n, block, r, inter):
    rng = np.random.default_rng(rank + heads_n)
    for new, ctx in (([1] * 7, [0, 5, 15, 16, 30, 63, 64]), ([70, 33, 200], [3, 0, 17])):
        slots, blocks = _slots(rng, new, ctx, block)
        slots[1], slots[-1] = -1, blocks * block + 2
        t = len(slots)
        g = torch.Generator(device=cuda).manual_seed(t)
        q = torch.randn((t, heads_n, rope + 128), generator=g, device=cuda).bfloat16()[:, :, 128:]
        kv = (3 * torch.randn((t, rank + rope), generator=g, device=cuda)).bfloat16()
        pos = torch.randint(0, 1 << 17, (t,), generator=g, device=cuda)
        freq = rotary_frequencies(r, 1e4, device=cuda)[0]
        angle = heads.phases(f64(pos), f64(freq))
        at = torch.from_numpy(slots).to(cuda)
        real = np.flatnonzero((slots >= 0) & (slots < blocks * block))
        for weight, eps, offset in ((torch.randn(rank, generator=g, device=cuda).bfloat16(), 1e-6, 0.0),
                                    (torch.randn(rank + 1, generator=g, device=cuda)[1:], 1e-5, 1.0), (None, None, 0.0)):
            c = MLALatentCache(blocks, block, rank, rope, device=cuda)
            c.latent.normal_(generator=g)
            guards = guard_cache(c)
            before = c.latent.clone()
            out = mla_rotary_append(q, kv[:, :rank], kv[:, rank:], c, at, pos, freq, kv_weight=weight, eps=eps,
                                    weight_offset=offset, interleaved=inter, scale=0.75)
            assert_guards(guards, "mla_rotary_append")
            check(out, heads.turn(f64(q), angle, inter, 0.75), 16 * U * size(f64(q), r // 2, inter, 0.75), "q_pe")
            x = f64(kv)
            # (a lane adds up to 24 squares here, 8 more than headcase.py counts: 4 u after the root)
            c_want = x[:, :rank] if eps is None else heads.norm(x[:, :rank], f64(weight), eps, offset)
            pe = heads.turn(x[:, None, rank:], angle, inter, 0.75)[:, 0]
            rows = c.latent.view(-1, rank + rope)
            check(rows[slots[real], :rank], c_want[real], 44 * U * np.abs(c_want[real]), "entries")
            check(rows[slots[real], rank:], pe[real], 16 * U * size(x[:, None, rank:], r // 2, inter, 0.75)[real, 0], "k_pe")
            rest = torch.ones(blocks * block, dtype=torch.bool, device=cuda)
            rest[slots[real]] = False
            assert torch.equal(rows[rest], before.view(-1, rank + rope)[rest])
            again = MLALatentCache(blocks, block, rank, rope, device=cuda)
            again.latent.copy_(before)
            mla_rotary_append(None, kv[:, :rank], kv[:, rank:], again, at, pos, freq, kv_weight=weight, eps=eps,
                              weight_offset=offset, interleaved=inter, scale=0.75)
            assert torch.equal(again.latent, c.latent)


def test_graph_replays(cuda):
    """Both appends captured, replayed over new inputs with eager work between."""
    rng = np.random.default_rng(8)
    slots, blocks = _slots(rng, [20, 1], [5, 16], 16)
    at = torch.from_numpy(slots).to(cuda)
    q, key, value, w, pos, freq = _inputs(cuda, 21, 4, 2, 64, 64, "dim")
    st = [x.contiguous().clone() for x in (q, key, value)]
    cache = _cache(cuda, blocks, 16, 2, 64, "fp8_e4m3")
    lat = MLALatentCache(blocks, 16, 512, 64, device=cuda)
    kv = torch.zeros((21, 576), device=cuda).bfloat16()
    norm = dict(q_weight=w[0], k_weight=w[1], eps=1e-6)

    def step(cache, lat, q, key, value, kv):
        a = rotary_append(q, key, value, cache, at, pos, freq, **norm)
        return a, mla_rotary_append(a, kv[:, :512], kv[:, 512:], lat, at, pos, freq, eps=1e-6)

    step(cache, lat, *st, kv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache, lat, *st, kv)
    for seed in range(3):
        new = _inputs(cuda, 21, 4, 2, 64, 64, "dim", seed=seed + 20)[:3]
        for a, b in zip(st, new):
            a.copy_(b)
        kv.normal_()
        start = _cache(cuda, blocks, 16, 2, 64, "fp8_e4m3", seed=seed)
        for a, b in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), (start.k, start.v, start.k_scale, start.v_scale)):
            a.copy_(b)
        lat.latent.zero_()
        graph.replay()
        torch.cuda.synchronize()
        other = MLALatentCache(blocks, 16, 512, 64, device=cuda)
        want = step(start, other, *new, kv)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]) and torch.equal(lat.latent, other.latent)
        for a, b in zip(_held(cache), _held(start)):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
def test_caches_of_more_than_2_31_elements(cuda, kv):
    """The last block of 1.1 million, beside the first one's, which stays; and the same of a latent cache."""
    blocks = 1_100_000
    c = PagedKVCache(blocks, 16, 1, 128, kv_dtype=kv, device=cuda)
    small = PagedKVCache(1, 16, 1, 128, kv_dtype=kv, device=cuda)
    for tokens in (5, 300):
        q, key, value, w, pos, freq = _inputs(cuda, tokens, 2, 1, 128, 128, "dim")
        slots = torch.full((tokens,), -1, device=cuda)
        slots[:5] = torch.arange(5, device=cuda)
        rotary_append(None, key, value, small, slots, pos, freq, k_weight=w[1], eps=1e-6)
        slots[:5] += (blocks - 1) * 16
        rotary_append(None, key, value, c, slots, pos, freq, k_weight=w[1], eps=1e-6)
        assert torch.equal(c.k[-1], small.k[0]) and torch.equal(c.v[-1], small.v[0])
        assert not c.k[0].any() and not c.v[0].any() and small.k[0].any()
    del c
    lat = MLALatentCache(240_000, 16, device=cuda)
    one = MLALatentCache(1, 16, device=cuda)
    kv_c, k_pe = torch.randn((3, 512), device=cuda).bfloat16(), torch.randn((3, 64), device=cuda).bfloat16()
    at, freq = torch.arange(3, device=cuda), rotary_frequencies(64, 1e4, device=cuda)[0]
    mla_rotary_append(None, kv_c, k_pe, one, at, at, freq, eps=1e-6)
    mla_rotary_append(None, kv_c, k_pe, lat, at + (240_000 - 1) * 16, at, freq, eps=1e-6)
    assert torch.equal(lat.latent[-1], one.latent[0]) and not lat.latent[0].any() and one.latent.any()


def test_latent_prompt_of_many_heads(cuda):
    """Heads of a token over several waves."""
    tokens = 4200
    g = torch.Generator(device=cuda).manual_seed(2)
    q = torch.randn((tokens, 70, 64), generator=g, device=cuda).bfloat16()
    kv = torch.randn((tokens, 576), generator=g, device=cuda).bfloat16()
    pos = torch.arange(tokens, device=cuda)
    freq = rotary_frequencies(64, 1e4, device=cuda)[0]
    c = MLALatentCache(264, 16, device=cuda)
    got = mla_rotary_append(q, kv[:, :512], kv[:, 512:], c, pos, pos, freq)
    angle = heads.phases(f64(pos), f64(freq))
    check(got, heads.turn(f64(q), angle), 16 * U * size(f64(q), 32, False, 1.0), "q_pe")
    rows = c.latent.view(-1, 576)[:tokens]
    assert torch.equal(rows[:, :512], kv[:, :512])
    x = f64(kv[:, None, 512:])
    check(rows[:, None, 512:], heads.turn(x, angle), 16 * U * size(x, 32, False, 1.0), "k_pe")


def test_no_tokens(cuda):
    c = _cache(cuda, 2, 16, 2, 64, "bf16")
    freq = rotary_frequencies(64, 1e4, device=cuda)[0]
    none = torch.zeros(0, dtype=torch.int64, device=cuda)
    x = torch.zeros((0, 2, 64), device=cuda).bfloat16()
    assert rotary_append(x, x, x, c, none, none, freq).shape == (0, 2, 64)


def test_refusals(cuda):
    q, key, value, w, pos, freq = _inputs(cuda, 4, 4, 2, 64, 64, "dim")
    c, lat = _cache(cuda, 2, 16, 2, 64, "bf16"), MLALatentCache(2, 16, 512, 64, device=cuda)
    slots = torch.arange(4, device=cuda)
    ok = dict(q=q, key=key, value=value, cache=c, slot_mapping=slots, positions=pos, inv_freq=freq)
    for bad in (dict(cache=lat), dict(key=key.float()), dict(key=key[:3]), dict(value=value[:, :1]),
                dict(slot_mapping=slots.int()), dict(slot_mapping=slots[:3]), dict(positions=None),
                dict(inv_freq=None, positions=None), dict(q_weight=w[0]), dict(weight_offset=1.0), dict(eps=0.0),
                dict(eps=1e-6, q_weight=w[0][:5]), dict(eps=1e-6, q_weight=w[0], k_weight=w[1].float()),
                dict(out=q.float()), dict(q=None, out=q), dict(q=q.cpu()), dict(q=q[:, :, :32]), dict(scale=float("nan")),
                dict(axes=torch.zeros(32, dtype=torch.int32, device=cuda)), dict(positions=pos[None])):
        with pytest.raises(ValueError):
            rotary_append(**{**ok, **bad})
    with pytest.raises(ValueError, match="gradient"):
        rotary_append(**{**ok, "key": key.detach().requires_grad_()})
    c.sleep()
    with pytest.raises(RuntimeError, match="asleep"):
        rotary_append(**ok)
    kv = torch.zeros((4, 576), device=cuda).bfloat16()
    ok = dict(q_pe=q, kv_c=kv[:, :512], k_pe=kv[:, 512:], cache=lat, slot_mapping=slots, positions=pos, inv_freq=freq)
    mla_rotary_append(**ok)
    for bad in (dict(cache=c), dict(kv_c=kv), dict(k_pe=kv[:3, 512:]), dict(kv_weight=torch.ones(512, device=cuda)),
                dict(eps=1e-6, kv_weight=torch.ones(64, device=cuda)), dict(eps=-1.0), dict(positions=pos[:2]),
                dict(eps=1e-6, kv_weight=torch.ones((1, 512), device=cuda)), dict(q_pe=None, out=q)):
        with pytest.raises(ValueError):
            mla_rotary_append(**{**ok, **bad})
