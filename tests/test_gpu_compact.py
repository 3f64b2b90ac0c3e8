"""The accepted path's move in the cache on the GPU: bit for bit the oracle's."""

import numpy as np
import pytest
import torch

from kvcase import assert_guards, bits_of, guard_cache, to_dev_bits
from oracle import fp8, paged, tree
from wavelet_amd import PagedKVCache

pytestmark = pytest.mark.gpu


def _case(cuda, seed, batch, hkv, d, bs, kv, ctx, new, depth, spread=(-8, -2)):
    rng = np.random.default_rng(seed)
    lens, n = rng.integers(ctx[0], ctx[1] + 1, batch), rng.integers(new[0], new[1] + 1, batch)
    blocks = -(-(lens + n) // bs)
    nb, width = int(blocks.sum()) + 2, max(int(blocks.max()), 1) + 1
    ids = rng.permutation(nb).astype(np.int32)
    bt = np.full((batch, width), -1, np.int32)
    at = 0
    for i, b in enumerate(blocks):
        bt[i, :b] = ids[at:at + b]
        at += b
    acc = np.array([rng.integers(0, min(depth, x) + 1) for x in n], np.int32)
    path = np.full((batch, depth), -1, np.int32)
    for i, a in enumerate(acc):
        if a:
            path[i, :a] = [0, *np.sort(rng.choice(np.arange(1, n[i]), a - 1, replace=False))]
    if kv == "bf16":
        k, v = paged.empty_cache(nb, bs, hkv, d)
        k[:], v[:] = (rng.integers(0, 65536, x.shape) for x in (k, v))  # any bits: a move changes none
        ks = vs = None
    else:
        k, v = paged.empty_cache(nb, bs, hkv, d, dtype=np.uint8)
        k[:], v[:] = (fp8.e4m3_encode((rng.normal(size=x.shape) * 60).astype(np.float32)) for x in (k, v))
        ks, vs = (np.exp2(rng.integers(*spread, size=(nb, hkv))).astype(np.float32) for _ in range(2))
    c = PagedKVCache(nb, bs, hkv, d, kv_dtype=kv, device=cuda)
    c.k.copy_(to_dev_bits(k, c.k.dtype, cuda))
    c.v.copy_(to_dev_bits(v, c.v.dtype, cuda))
    if ks is not None:
        c.k_scale.copy_(torch.from_numpy(ks))
        c.v_scale.copy_(torch.from_numpy(vs))
    return c, [k, v, ks, vs], bt, lens.astype(np.int32), path, acc


def _check(c, host, what):
    for name, x in zip(("k", "v", "k_scale", "v_scale"), host):
        if x is not None:
            np.testing.assert_array_equal(bits_of(getattr(c, name)), x, err_msg=f"{what}: {name}")


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("seed,batch,hkv,d,bs,ctx,new,depth", [
    (0, 1, 1, 64, 16, (0, 0), (1, 1), 1), (1, 9, 2, 128, 16, (0, 100), (0, 40), 8), (2, 64, 8, 128, 16, (65, 500), (16, 16), 8),
    (3, 5, 4, 64, 48, (0, 300), (60, 130), 64), (4, 7, 2, 128, 256, (0, 600), (100, 256), 64), (5, 33, 4, 128, 32, (1, 90), (9, 63), 12),
    (6, 4, 3, 64, 64, (63, 64), (64, 200), 40), (7, 300, 2, 64, 16, (0, 40), (2, 6), 5)])
def test_compact(cuda, kv, seed, batch, hkv, d, bs, ctx, new, depth):
    c, host, bt, lens, path, acc = _case(cuda, seed, batch, hkv, d, bs, kv, ctx, new, depth)
    g = guard_cache(c)
    args = [torch.from_numpy(x).to(cuda) for x in (bt, lens, path, acc)]
    c.compact(*args)
    tree.compact(*host, bt, lens, path, acc)
    _check(c, host, f"{kv} {seed}")
    assert_guards(g, "cache")


def test_compact_scales_far_apart(cuda):
    """Blocks whose scales differ by up to 2^24: tokens round to nothing, blocks grow, blocks start afresh."""
    c, host, bt, lens, path, acc = _case(cuda, 11, 40, 4, 128, 16, "fp8_e4m3", (0, 60), (10, 60), 20, spread=(-14, 10))
    c.compact(*[torch.from_numpy(x).to(cuda) for x in (bt, lens, path, acc)])
    tree.compact(*host, bt, lens, path, acc)
    _check(c, host, "far apart")


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
def test_compact_keeps_chains_and_places_without_blocks(cuda, kv):
    c, host, bt, lens, path, acc = _case(cuda, 5, 6, 2, 64, 16, kv, (10, 60), (20, 30), 8)
    chain = np.tile(np.arange(8, dtype=np.int32), (6, 1))
    dev = lambda *x: [torch.from_numpy(np.ascontiguousarray(y)).to(cuda) for y in x]  # noqa: E731
    c.compact(*dev(bt, lens, chain, acc * 0 + 8))
    _check(c, host, "a chain")
    # sequences without a block at the places: nothing moves, and the others' do
    bad = bt.copy()
    bad[1::2] = [[-1], [10**6], [-7]]
    c.compact(*dev(bad, lens, path, acc))
    keep = [x for x in range(6) if x % 2 == 0]
    tree.compact(*host, bt[keep], lens[keep], path[keep], acc[keep])
    _check(c, host, "no blocks")
    # past the table's width, and no sequences at all
    c.compact(*dev(bt[:, :1], lens + 1000, path, acc))
    c.compact(*dev(bt[:0], lens[:0], path[:0], acc[:0]))
    _check(c, host, "outside")


def test_compact_refusals(cuda):
    c, _, bt, lens, path, acc = _case(cuda, 5, 6, 2, 64, 16, "bf16", (10, 60), (20, 30), 8)
    a = [torch.from_numpy(x).to(cuda) for x in (bt, lens, path, acc)]
    for bad in ((a[0].long(), *a[1:]), (a[0], a[1].long(), *a[2:]), (*a[:2], a[2].long(), a[3]), (*a[:2], a[2][:3], a[3]),
                (*a[:2], a[2][:, :0], a[3]), (*a[:2], a[2].repeat(1, 9), a[3]), (*a[:3], a[3][:2]), (*a[:3], a[3].cpu())):
        with pytest.raises(ValueError):
            c.compact(*bad)
    c.sleep()
    with pytest.raises(RuntimeError):
        c.compact(*a)
