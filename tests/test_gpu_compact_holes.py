"""Accepted paths over tables with entries that are no blocks, in their midst: bit for bit the oracle's.

What loses its old or its new place stays behind; a block's other tokens are one append, as ever.
"""

import numpy as np
import pytest
import torch

from kvcase import assert_guards, guard_cache
from oracle import tree
from test_gpu_compact import _case, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("seed,batch,hkv,d,bs,ctx,new,depth,holes", [
    (0, 20, 2, 64, 16, (0, 40), (60, 130), 20, 0.3), (1, 33, 4, 128, 16, (1, 90), (100, 250), 64, 0.15),
    (2, 9, 1, 128, 32, (0, 60), (200, 256), 40, 0.3), (3, 12, 2, 64, 16, (0, 40), (60, 130), 30, 0.7)])
def test_tables_with_holes(cuda, kv, seed, batch, hkv, d, bs, ctx, new, depth, holes):
    c, host, bt, lens, path, acc = _case(cuda, seed, batch, hkv, d, bs, kv, ctx, new, depth)
    rng = np.random.default_rng(100 + seed)
    hole = rng.random(bt.shape) < holes
    bt[hole] = rng.choice([-1, -9, len(host[0]), 2**31 - 1], int(hole.sum()))
    g = guard_cache(c)
    c.compact(*(torch.from_numpy(x).to(cuda) for x in (bt, lens, path, acc)))
    tree.compact(*host, bt, lens, path, acc)
    _check(c, host, f"{kv} {seed}")
    assert_guards(g, "cache")


def test_a_hole_splits_no_run(cuda):
    """New places 11, 12, 13 .. of one block, 12's token from a block that is none: the others are one append."""
    c, host, bt, _, _, _ = _case(cuda, 9, 6, 2, 128, 16, "fp8_e4m3", (10, 10), (60, 60), 8)
    lens, acc = np.full(6, 10, np.int32), np.full(6, 5, np.int32)
    path = np.tile(np.array([0, 2, 9, 25, 41], np.int32), (6, 1))  # positions 10, 12, 19, 35, 51 to 10 .. 14
    bt[:, 1] = -1  # 19 was there
    c.compact(*(torch.from_numpy(x).to(cuda) for x in (bt, lens, path, acc)))
    tree.compact(*host, bt, lens, path, acc)
    _check(c, host, "a hole")


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
def test_path_entries_that_name_no_node(cuda, kv):
    c, host, bt, lens, path, acc = _case(cuda, 6, 8, 2, 64, 16, kv, (0, 40), (30, 60), 12)
    path[::2, 3] = -1
    path[1::2, 5] = 2**31 - 1
    c.compact(*(torch.from_numpy(x).to(cuda) for x in (bt, lens, path, acc)))
    tree.compact(*host, bt, lens, path, acc)
    _check(c, host, "no nodes")
