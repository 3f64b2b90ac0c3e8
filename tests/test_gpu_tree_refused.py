"""Rows of sequences that a step refused: zeros, however the attention is launched."""

import pytest
import torch

from kvcase import bits_of, check_attention
from oracle import paged
from test_gpu_tree import Case
from wavelet_amd import KVPool, paged_tree_gqa
from wavelet_amd.plan import TreeStep

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("longest", [500, 3000])  # one workgroup per row group; the steps shared
def test_rows_past_max_query_len(cuda, longest):
    """A sequence of length 0 (refused, for its 200 nodes say) with more rows than max_query_len: all are zeros."""
    c = Case(cuda, f"refused{longest}", 8, 2, 128, 16, [40, 20, longest], [64, 200, 9], words=4)
    q, cache, bt, sl, cu, mask, scale = c.args()
    c._append(c.kn, c.vn, c.slots)
    c.upload()
    sl[1] = 0
    lens = c.lens.copy()
    lens[1] = 0
    out = torch.full_like(q, float("nan"))
    paged_tree_gqa(q, cache, bt, sl, cu, mask, scale, max_query_len=64, max_seq_len=longest + 9, out=out)
    assert (out[64:264] == 0).all()
    check_attention(paged.bf16_to_f32(bits_of(out)), c.ref(seq_lens=lens), "the others")


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("longest", [500, 3000])
@pytest.mark.parametrize("bound", [1, 64, 100])
def test_rows_past_max_query_len_of_others(cuda, kv, longest, bound):
    """A bound that is too low costs time, not rows."""
    c = Case(cuda, f"low{kv}{longest}", 8, 2, 64, 16, [40, longest, 0, 90], [200, 70, 0, 1], kv)
    out = paged_tree_gqa(*c.args(), **c.appended(), max_query_len=bound, max_seq_len=longest + 240)
    c.append_host()
    check_attention(paged.bf16_to_f32(bits_of(out)), c.ref(), "low bound")


@pytest.mark.parametrize("max_seq_len", [512, 4096])
def test_a_step_with_too_many_nodes(cuda, max_seq_len):
    """TreeStep: a sequence refused for its 200 nodes of 64; its rows of `out` hold nothing of the step before."""
    hq, hkv, d = 8, 2, 64
    pool = KVPool(1, 600, 16, hkv, d, device=cuda, max_model_len=max_seq_len)
    for i in range(2):
        pool.blocks.allocate(i, range(30))
    state = pool.lend([0, 1], 40)
    T = 240
    q, out = (torch.randn((T, hq, d), device=cuda).to(BF16) for _ in range(2))
    k, v = (torch.randn((T, hkv, d), device=cuda).to(BF16) for _ in range(2))
    chain = torch.arange(T, dtype=torch.int32, device=cuda) - 1
    tokens = torch.zeros(T, dtype=torch.int64, device=cuda)
    new = torch.tensor([200, 20], dtype=torch.int32, device=cuda)
    step = TreeStep(pool.layers, [q], [k], [v], [out], state, new, chain, tokens, tokens, d ** -0.5, 64, max_seq_len, 8)
    step.begin()
    step.run()
    assert int(step.maps.refused) == 1 and step.maps.context_lens.tolist() == [0, 50]
    assert (out[:200] == 0).all() and (out[200:220] != 0).any(-1).all()
