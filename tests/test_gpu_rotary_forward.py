"""Forward-mode derivatives of the rotation: the tangents are turned as the values are.

The rotation is linear, so a tangent's result is the call's on the tangent, bit for bit.
"""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from wavelet_amd import apply_rotary, rotary_frequencies

pytestmark = pytest.mark.gpu


def _case(cuda, dtype=torch.float32):
    g = torch.Generator(device=cuda).manual_seed(5)
    rnd = lambda h: torch.randn((9, h, 64), generator=g, device=cuda).to(dtype)  # noqa: E731
    return rnd(4), rnd(2), rnd(4), rnd(2), torch.arange(9, device=cuda) * 77, rotary_frequencies(48, device=cuda)[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("with_q,with_k", [(True, True), (True, False), (False, True)])
def test_tangents(cuda, dtype, inter, with_q, with_k):
    q, k, tq, tk, pos, freq = _case(cuda, dtype)
    yq, yk = apply_rotary(q, k, pos, freq, interleaved=inter, scale=1.25)
    wq, wk = apply_rotary(tq, tk, pos, freq, interleaved=inter, scale=1.25)
    with fwd.dual_level():
        a = fwd.make_dual(q, tq) if with_q else q
        b = fwd.make_dual(k, tk) if with_k else k
        got = [fwd.unpack_dual(x) for x in apply_rotary(a, b, pos, freq, interleaved=inter, scale=1.25)]
    for (primal, tangent), y, w, given in zip(got, (yq, yk), (wq, wk), (with_q, with_k)):
        assert torch.equal(primal, y)
        if given:
            assert torch.equal(tangent, w)
        else:
            assert tangent is None or not tangent.any()


def test_tangents_without_k_of_strided_rows_and_turned_back(cuda):
    q, _, tq, _, pos, freq = _case(cuda)
    t = tq.transpose(1, 2).contiguous().transpose(1, 2)  # last dim strided
    with fwd.dual_level(), torch.no_grad():
        y, none = apply_rotary(fwd.make_dual(q, t), None, pos, freq, inverse=True)
        assert none is None and torch.equal(fwd.unpack_dual(y).tangent, apply_rotary(tq, None, pos, freq, inverse=True)[0])
        plain, _ = apply_rotary(q, None, pos, freq, inverse=True)  # no tangent at this level
        assert fwd.unpack_dual(plain).tangent is None and torch.equal(plain, fwd.unpack_dual(y).primal)


def test_tangent_of_a_gradient(cuda):
    """Forward over reverse: y -> R q, loss = sum (R q)^3, its gradient R^T 3 (R q)^2, that one's derivative along t
    R^T (6 (R q) (R t)). float32: a few roundings of values below 2^9."""
    q, _, tq, _, pos, freq = _case(cuda)
    q.requires_grad_()
    with fwd.dual_level():
        y, _ = apply_rotary(fwd.make_dual(q, tq), None, pos, freq)
        (g,) = torch.autograd.grad((y ** 3).sum(), q)
        got = fwd.unpack_dual(g).tangent
    with torch.no_grad():
        rq, rt = (apply_rotary(x, None, pos, freq)[0] for x in (q, tq))
        want = apply_rotary(6 * rq * rt, None, pos, freq, inverse=True)[0]
    assert got is not None
    torch.testing.assert_close(got, want, rtol=0, atol=2.0 ** 9 * 2.0 ** -20)


def test_out_takes_no_tangents(cuda):
    q, k, tq, _, pos, freq = _case(cuda)
    before = q.clone()
    with fwd.dual_level():
        with pytest.raises(ValueError, match="out and gradients"):
            apply_rotary(fwd.make_dual(q, tq), k, pos, freq, out=(q, k))
    assert torch.equal(q, before)


def test_gradient_of_a_tangent(cuda):
    """Reverse over forward: q = w x along v has the tangent R (w v), whose product with c has the gradient
    v R^T c in w. float32: a few roundings of values below 2^6."""
    x, _, v, _, pos, freq = _case(cuda)
    w, c = torch.randn_like(x).requires_grad_(), torch.randn_like(x)
    for k in (None, torch.randn_like(x)):
        with fwd.dual_level():
            y, _ = apply_rotary(w * fwd.make_dual(x, v), k, pos, freq)
            (g,) = torch.autograd.grad((fwd.unpack_dual(y).tangent * c).sum(), w)
        want = v * apply_rotary(c, None, pos, freq, inverse=True)[0]
        torch.testing.assert_close(g, want, rtol=0, atol=2.0 ** 6 * 2.0 ** -21)
