"""The oracle of a step of drafted tokens against what it must agree with, and the refusals of the Python
entry points (CPU)."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import fp8, paged, tree
from test_abi import host_only
from wavelet_amd import BlockManager, _lib, accept_tree, apply_rotary, extend_tables, rotary_frequencies


def _rng(seed):
    return np.random.default_rng(seed)


def test_rotation_keeps_norms_and_its_inverse_undoes_it():
    x = _rng(1).normal(size=(5, 3, 32))
    pos, freq = np.array([0, 1, 7, 100000, -3]), 1e4 ** (-np.arange(8) / 8)
    for inter in (False, True):
        y = tree.rotary(x, pos, freq, interleaved=inter, scale=2.0)
        np.testing.assert_allclose(np.square(y[..., :16]).sum(-1), 4 * np.square(x[..., :16]).sum(-1))
        np.testing.assert_array_equal(y[..., 16:], x[..., 16:])
        np.testing.assert_allclose(tree.rotary(y, pos, freq, interleaved=inter, scale=0.5, inverse=True), x, atol=1e-12)
        np.testing.assert_array_equal(tree.rotary(x[:1], pos[:1], freq, interleaved=inter), x[:1])
    # a query's product with a key depends on the distance of their positions alone
    q, k = x[:1], x[1:2]
    dot = [(tree.rotary(q, [p + 9], freq) * tree.rotary(k, [p], freq)).sum() for p in (0, 5, 4000)]
    np.testing.assert_allclose(dot, dot[0])


def test_tables_of_single_tokens_are_the_block_managers():
    bm = BlockManager(64, 16)
    lens = [0, 15, 16, 33]
    for i, n in enumerate(lens):
        bm.allocate(i, np.arange(n) + 1000 * i)
    bt, sl = bm.tables(range(4), width=4)
    held = [len(bm.blocks_of(i)) for i in range(4)]
    free = [b for b in range(64) if bm.ref_count(b) == 0]
    out = tree.extend_tables(bt, held, sl, [1] * 4, free, 0, 16, 6)
    slots, cow = bm.append_slots(range(4))
    assert cow == []
    np.testing.assert_array_equal(out["slot_mapping"], [*slots, -1, -1])
    np.testing.assert_array_equal(out["block_table"], bm.tables(range(4), width=4)[0])
    assert out["taken"] == 2 and out["refused"] == 0
    np.testing.assert_array_equal(out["context_lens"], sl + 1)


def test_refused_sequences_get_nothing():
    bt = np.full((4, 2), -1, np.int32)
    # 40 tokens pass two blocks of 16; 20 need two of three blocks; 17 more than the one left; 3 fit no more rows
    out = tree.extend_tables(bt, [0] * 4, [0] * 4, [40, 20, 17, 3], [5, 6, 7], 0, 16, 79)
    np.testing.assert_array_equal(out["context_lens"], [0, 20, 0, 0])
    np.testing.assert_array_equal(out["cu_seqlens_q"], [0, 40, 60, 77, 79])
    assert out["refused"] == 3 and out["taken"] == 2
    np.testing.assert_array_equal(out["block_table"], [[-1, -1], [5, 6], [-1, -1], [-1, -1]])


def test_accepted_path_follows_the_first_child_that_agrees():
    parents = np.array([-1, 0, 0, 0, 2, 2, 4], np.int32)
    draft = np.array([9, 5, 7, 7, 1, 3, 8])
    target = np.array([7, 0, 3, 0, 0, 4, 0])
    acc, path, nxt, lens = tree.accept_tree(draft, parents, target, [0, 7], [10], [17], 5)
    assert acc[0] == 3 and nxt[0] == 4 and lens[0] == 13
    np.testing.assert_array_equal(path[0], [0, 2, 5, -1, -1])  # node 2 before its equal 3
    acc, path, nxt, _ = tree.accept_tree(draft, parents, target, [0, 7], [10], [17], 2)
    assert acc[0] == 2 and nxt[0] == 3


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_move_is_gather_then_append(kv):
    rng, bs, h, d = _rng(3), 16, 2, 64
    bt = np.array([[3, 0, 5], [1, 4, 2]], np.int32)
    lens, acc = np.array([10, 30]), np.array([4, 5])
    path = np.array([[0, 2, 3, 9, -1], [0, 1, 2, 3, 4]], np.int32)
    dt = np.uint16 if kv == "bf16" else np.uint8
    k, v = paged.empty_cache(6, bs, h, d, dtype=dt)
    if kv == "bf16":
        k[:] = paged.f32_to_bf16(rng.normal(size=k.shape))
        v[:] = paged.f32_to_bf16(rng.normal(size=v.shape))
        ks = vs = None
    else:
        k[:], v[:] = (fp8.e4m3_encode(rng.normal(size=x.shape).astype(np.float32) * 20) for x in (k, v))
        ks, vs = (np.exp2(rng.integers(-6, -2, size=(6, h))).astype(np.float32) for _ in range(2))
    before = [None if x is None else x.copy() for x in (k, v, ks, vs)]
    gk, gv = paged.gather(k, v, bt, [22, 35])
    tree.compact(k, v, ks, vs, bt, lens, path, acc)
    # the second sequence's path keeps its place; the first moves nodes 2, 3, 9 behind node 0
    for x, y in zip(before, (k, v, ks, vs)):
        if x is not None:
            np.testing.assert_array_equal(x[[1, 4, 2]], y[[1, 4, 2]])
    hk, hv = paged.gather(k, v, bt, [14, 35])
    if kv == "bf16":
        np.testing.assert_array_equal(hk[:14], gk[[*range(11), 12, 13, 19]])
        np.testing.assert_array_equal(hv[:14], gv[[*range(11), 12, 13, 19]])
    else:
        got = fp8.dequantize(hk[:14], ks[bt[0, np.arange(14) // bs]][:, :, None])
        src = np.array([*range(11), 12, 13, 19])
        want = fp8.dequantize(gk[src], before[2][bt[0, src // bs]][:, :, None])
        # a value coded again is off by half a step: 2^-4 of itself, or of the least normal number at the scale
        s = ks[bt[0, np.arange(14) // bs]][:, :, None]
        assert (np.abs(got - want) <= 2.0 ** -4 * np.abs(want) + 2.0 ** -10 * s).all()


def test_chain_attention_is_the_prefills():
    rng = _rng(4)
    kv = rng.normal(size=(2, 8, 16, 2, 8))
    q = rng.normal(size=(7, 4, 8))
    bt, lens, cu = np.array([[0, 1, 2], [5, 3, 7]], np.int32), [40, 3], [0, 4, 7]
    masks = np.concatenate([tree.masks(np.arange(-1, n - 1), 1) for n in (4, 3)])
    got = tree.tree_gqa(q, *kv, bt, lens, cu, masks, 0.3)
    np.testing.assert_allclose(got, paged.prefill_gqa(q, *kv, bt, lens, cu, 0.3), atol=1e-12)


def test_masks_hold_the_ancestors():
    m = tree.masks([-1, 0, 0, 2, 9, -5, 3], 1)[:, 0]
    assert m.tolist() == [1, 3, 5, 13, 16, 32, 77]  # 9 and -5 are no earlier nodes


# ---------------------------------------------------------------------------- frequencies and refusals

@pytest.mark.parametrize("name,cfg", [
    ("default", {}), ("linear", dict(factor=4.0)),
    ("dynamic", dict(factor=2.0)),
    ("llama3", dict(factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192)),
    ("yarn", dict(factor=16.0, original_max_position_embeddings=4096)),
    ("yarn", dict(factor=40.0, original_max_position_embeddings=4096, mscale=1.0, mscale_all_dim=0.8, beta_fast=16.0)),
    ("yarn", dict(factor=4.0, original_max_position_embeddings=32768, attention_factor=1.5))])
def test_frequencies_are_transformers(name, cfg):
    """Against the same scalings of the transformers library (float32 there: 2^-20 covers its powers and products)."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    scaling = dict(rope_type=name, rope_theta=500000.0, **cfg)
    c = LlamaConfig(hidden_size=256, num_attention_heads=2, head_dim=128, max_position_embeddings=8192,
                    rope_theta=500000.0, rope_scaling=dict(scaling), rope_parameters=dict(scaling))
    if name == "default":
        want, gain = 500000.0 ** (-torch.arange(0, 128, 2).double() / 128), 1.0
    else:
        more = dict(seq_len=20000) if name == "dynamic" else {}
        want, gain = ROPE_INIT_FUNCTIONS[name](c, "cpu", **more)
    if name == "dynamic":
        scaling.update(max_length=20000, original_max_position_embeddings=8192)
    got, scale = rotary_frequencies(128, 500000.0, scaling=None if name == "default" else scaling, device="cpu")
    assert got.dtype == torch.float64
    torch.testing.assert_close(got, want.double(), rtol=2.0 ** -20, atol=0)
    assert scale == pytest.approx(gain, rel=1e-6)


def test_frequency_refusals():
    with pytest.raises(ValueError):
        rotary_frequencies(63, device="cpu")
    with pytest.raises(ValueError, match="factor"):
        rotary_frequencies(64, scaling=dict(rope_type="linear"), device="cpu")
    with pytest.raises(NotImplementedError):
        rotary_frequencies(64, scaling=dict(rope_type="longrope"), device="cpu")


def test_entry_points_need_the_gpu():
    t = torch.zeros((2, 1, 8))
    with pytest.raises(ValueError, match="GPU"):
        apply_rotary(t, None, torch.zeros(2, dtype=torch.int64), torch.ones(2, dtype=torch.float64))
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        extend_tables(torch.zeros((2, 3), dtype=torch.int32), i, i, i, i, i[:1], 16, 4)
    with pytest.raises(ValueError, match="GPU"):
        accept_tree(i.long(), i, i.long(), torch.zeros(3, dtype=torch.int32), i, i, 4)


P = 4096  # a fake, aligned device pointer: every call below is refused before a launch


def _rotary(**kw):
    a = dict(dtype=1, q=P, qt=256, qh=64, qo=P, qot=256, qoh=64, hq=4, k=P, kt=64, kh=64, ko=P, kot=64, koh=64, hk=1,
             d=64, pos=P, freq=P, r=64, inter=0, inv=0, scale=1.0, n=2, stream=None)
    a.update(kw)
    return _lib.load().wkv_rotary(*a.values())


@host_only
@pytest.mark.parametrize("kw", [dict(dtype=3), dict(d=63), dict(d=514), dict(r=66), dict(r=0), dict(r=3), dict(q=None),
                                dict(q=P + 1), dict(kt=-1), dict(pos=None), dict(freq=P + 4), dict(n=-1), dict(hq=-1),
                                dict(scale=float("inf"))])
def test_rotary_refusals(kw):
    assert _rotary(**kw) == _lib.WKV_ERR_INVALID


def _tables(**kw):
    a = dict(bt=P, stride=8, width=8, held=P, lens=2 * P, new=3 * P, batch=2, bs=16, free=P, nfree=4, taken=P, rows=8,
             parents=P, words=1, held_out=P, taken_out=P, context=4 * P, cu=P, slots=P, pos=P, mask=P, refused=P,
             stream=None)
    a.update(kw)
    return _lib.load().wkv_extend_tables(*a.values())


@host_only
@pytest.mark.parametrize("kw", [dict(batch=0), dict(batch=2049), dict(stride=7), dict(width=0), dict(bs=0), dict(rows=-1),
                                dict(words=5), dict(parents=None), dict(mask=None), dict(free=None), dict(taken=None),
                                dict(context=2 * P), dict(context=3 * P), dict(slots=None), dict(bt=None)])
def test_tables_refusals(kw):
    assert _tables(**kw) == _lib.WKV_ERR_INVALID


def _desc(**kw):
    base = dict(k=P, v=P, k_scale=None, v_scale=None, num_blocks=4, block_size=16, num_kv_heads=2, head_dim=128,
                kv_dtype=_lib.WKV_KV_BF16)
    base.update(kw)
    return _lib.WkvCache(**base)


def _tree(desc=None, **kw):
    a = dict(key=None, kt=0, kh=0, value=None, vt=0, vh=0, slots=None, n=0, q=P, qt=512, qh=128, out=P, ot=512, oh=128,
             hq=4, cu=P, lens=P, bt=P, stride=8, width=8, batch=2, mq=8, ms=100, mask=P, words=1, scale=1.0, ws=None,
             wsb=0, sinks=None, stream=None)
    a.update(kw)
    return _lib.load().wkv_tree_gqa(ctypes.byref(desc or _desc()), *a.values())


@host_only
@pytest.mark.parametrize("kw", [dict(hq=5), dict(q=None), dict(q=P + 8), dict(qt=511), dict(out=None), dict(ot=510),
                                dict(cu=None), dict(stride=7), dict(mq=-1), dict(mask=None), dict(mask=P + 4),
                                dict(words=0), dict(words=5), dict(scale=float("nan")), dict(sinks=P + 2),
                                dict(batch=65536), dict(mq=1 << 24), dict(ms=100000, width=8192, stride=8192, ws=P, wsb=64)])
def test_tree_refusals(kw):
    assert _tree(**kw) == _lib.WKV_ERR_INVALID


@host_only
def test_tree_refuses_other_heads_and_bad_workspace_geometry():
    assert _tree(_desc(head_dim=96)) == _lib.WKV_ERR_UNSUPPORTED
    size = _lib.load().wkv_tree_workspace_size
    assert size(2, 0, 2, 5, 128, 8, 100) == -1 and size(2, 0, 2, 4, 96, 8, 100) == -1 and size(2, 3, 2, 4, 128, 8, 9) == -1
    assert size(0, 0, 2, 4, 128, 8, 100) == 0 and size(1, 0, 2, 4, 128, 8, 100000) > 0


@host_only
@pytest.mark.parametrize("kw", [dict(depth=0), dict(depth=65), dict(path=None), dict(stride=7), dict(batch=70000),
                                dict(accepted=None)])
def test_compact_refusals(kw):
    a = dict(bt=P, stride=8, width=8, lens=P, path=P, depth=4, accepted=P, batch=2, stream=None)
    a.update(kw)
    assert _lib.load().wkv_compact(ctypes.byref(_desc()), *a.values()) == _lib.WKV_ERR_INVALID


@host_only
@pytest.mark.parametrize("kw", [dict(depth=0), dict(depth=65), dict(draft=None), dict(batch=-1), dict(out=None),
                                dict(rows=-1), dict(rows=2**31)])
def test_accept_refusals(kw):
    a = dict(draft=P, parents=P, target=P, rows=9, cu=P, lens=P, context=P, batch=2, depth=4, acc=P, path=P, nxt=P, out=P,
             stream=None)
    a.update(kw)
    assert _lib.load().wkv_accept_tree(*a.values()) == _lib.WKV_ERR_INVALID
