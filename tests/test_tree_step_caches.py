"""What TreeStep refuses before it looks at anything else (CPU)."""

import pytest
import torch

from wavelet_amd import KVPool
from wavelet_amd.plan import TreeStep


def test_mla_caches_are_refused():
    """A latent cache has neither tree attention nor a move; its blocks can be lent for steps of known slots."""
    pool = KVPool(1, 8, 16, mla=True, device="cpu")
    pool.blocks.allocate(0, range(20))
    state = pool.lend([0], 2)
    t = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="PagedKVCache"):
        TreeStep(pool.layers, [t], [t], [t], [t], state, t[:1].int(), t.int(), t, t, 1.0, 64, 128, 8)
