"""Drafted attention of sequences longer than what the call allows: max_seq_len, or the width of the table.

Tokens past the limit are attended by no row; the others, context and drafted, as ever. The oracle is given a
table without blocks past the limit, a multiple of the block size here.
"""

import pytest

from kvcase import bits_of, check_attention
from oracle import paged
from test_gpu_tree import Case
from wavelet_amd import paged_tree_gqa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("ctx,new,limit", [
    ([300, 90], [20, 33], 304),             # the limit is among the drafted tokens
    ([300, 90, 7], [64, 9, 1], 240),        # before them: context is cut, no drafted token is seen
    ([2500, 40, 900], [17, 64, 3], 2512),   # contexts that may be cut over workgroups
    ([4000, 40, 900], [130, 64, 3], 2032),  # a limit that is no multiple of a step's keys
    ([700, 800], [16, 16], 832)])           # a length that is one
def test_keys_past_the_limit(cuda, kv, ctx, new, limit):
    c = Case(cuda, f"longest{kv}{ctx[0]}{limit}", 8, 2, 128, 16, ctx, new, kv)
    c._append(c.kn, c.vn, c.slots)
    c.upload()
    bt = c.w.block_tables.copy()
    bt[:, limit // 16:] = -1
    ref = c.ref(block_table=bt)
    q, cache, table, sl, cu, mask, scale = c.args()
    out = paged_tree_gqa(q, cache, table, sl, cu, mask, scale, max_seq_len=limit)
    check_attention(paged.bf16_to_f32(bits_of(out)), ref, "max_seq_len")
    out = paged_tree_gqa(q, cache, table[:, :limit // 16], sl, cu, mask, scale)
    check_attention(paged.bf16_to_f32(bits_of(out)), ref, "the table's width")
