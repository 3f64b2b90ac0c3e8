"""A rotation into given tensors counts as a write for autograd: what was saved of them before is stale."""

import pytest
import torch

from wavelet_amd import apply_rotary, rotary_frequencies

pytestmark = pytest.mark.gpu


def test_in_place_marks_what_autograd_saved(cuda):
    pos, freq = torch.arange(5, device=cuda), rotary_frequencies(64, device=cuda)[0]
    w = torch.randn((5, 2, 64), device=cuda, requires_grad=True)
    q, k = torch.randn((5, 2, 64), device=cuda), torch.randn((5, 1, 64), device=cuda)
    loss = (w * q).sum()  # the gradient of w is q, saved
    apply_rotary(q, k, pos, freq, out=(q, k))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    k2 = torch.randn((5, 2, 64), device=cuda)
    loss = (w * k2).sum()
    apply_rotary(q, k2, pos, freq, out=(q, k2))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_out_that_needs_a_gradient_is_refused(cuda):
    pos, freq = torch.arange(5, device=cuda), rotary_frequencies(64, device=cuda)[0]
    q, k = torch.randn((5, 2, 64), device=cuda), torch.randn((5, 1, 64), device=cuda)
    for out in ((q.clone().requires_grad_(), k), (q, k.clone().requires_grad_())):
        with pytest.raises(ValueError, match="out and gradients"):
            apply_rotary(q, k, pos, freq, out=out)
        with torch.no_grad():
            apply_rotary(q, k, pos, freq, out=out)
    with torch.inference_mode():  # tensors without versions
        x = q.clone()
        apply_rotary(x, None, pos, freq, out=(x, None))
    assert torch.equal(x, apply_rotary(q, None, pos, freq)[0])
