"""Drafted attention without a sequence: its tokens are appended all the same, as prefill_gqa does it."""

import pytest
import torch

from wavelet_amd import PagedKVCache, paged_tree_gqa, prefill_gqa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("batch", [0, 2])
def test_rows_of_no_sequence_are_appended(cuda, kv, batch):
    caches = [PagedKVCache(4, 16, 2, 64, kv_dtype=kv, device=cuda) for _ in range(2)]
    k, v, q = (torch.randn((5, h, 64), device=cuda).to(torch.bfloat16) for h in (2, 2, 4))
    slots = torch.tensor([17, 18, 19, -1, -1], device=cuda)
    i = torch.zeros(batch + 1, dtype=torch.int32, device=cuda)
    bt = torch.zeros((batch, 3), dtype=torch.int32, device=cuda)
    new = dict(key=k, value=v, slot_mapping=slots)
    out = torch.full_like(q, 7.0)
    paged_tree_gqa(q, caches[0], bt, i[:batch], i, torch.zeros((5, 1), dtype=torch.int64, device=cuda), 0.125, out=out, **new)
    prefill_gqa(q, caches[1], bt, i[:batch], i, 0.125, **new)
    assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)
    assert caches[0].k.any() and (out == 7).all()
