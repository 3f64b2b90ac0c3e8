"""Lent blocks taken back while steps on another stream are still running."""

import pytest
import torch

from wavelet_amd import KVPool

pytestmark = pytest.mark.gpu


def test_settle_waits_for_steps_on_other_streams(cuda):
    pool = KVPool(1, 64, 16, 2, 64, device=cuda)
    pool.blocks.allocate("a", range(30))
    state = pool.lend(["a"], 8)
    new = torch.tensor([20], dtype=torch.int32, device=cuda)
    x = torch.randn((4096, 4096), device=cuda)
    state.extend(new * 0, 20)  # (the first launch of a kernel is slow)
    torch.cuda.synchronize()
    s = torch.cuda.Stream(cuda)
    with torch.cuda.stream(s):
        for _ in range(60):  # some milliseconds of work ahead of the step
            y = x @ x
        m = state.extend(new, 20)
        state.seq_lens.copy_(m.context_lens)
    pool.settle(state)
    assert pool.blocks.seq_len("a") == 50 and len(pool.blocks.blocks_of("a")) == 4
    assert torch.isfinite(y).all()
