"""Rotary positions on the GPU against the float64 oracle.

Tolerance: the result's rounding, half a step of its type (eps / 2 of the value), and the float32
arithmetic before it: the reduced angle is off by at most 2^-25 of half a turn (2^-23 of a radian), each sine and
cosine by two units (2^-23), their factor, the two products and the sum by half a unit each:
together below 16 x 2^-24 of scale (|x_a| + |x_b|).
"""

import numpy as np
import pytest
import torch

from oracle import tree
from wavelet_amd import apply_rotary, rotary_frequencies

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _check(got, x, pos, freq, inter, scale=1.0, inverse=False):
    x = x.detach().double().cpu().numpy()
    f = freq.cpu().numpy()
    want = tree.rotary(x, pos.cpu().numpy(), f, interleaved=inter, scale=scale, inverse=inverse)
    half = len(f)
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if inter else (i, i + half)
    size = np.zeros_like(x)
    size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * np.abs(want) + 16 * 2.0 ** -24 * abs(scale) * size + fi.smallest_normal * fi.eps
    err = np.abs(got.detach().double().cpu().numpy() - want)
    assert (err <= tol).all(), f"off by {(err / tol).max():.3f} of the tolerance"
    np.testing.assert_array_equal(got.detach().double().cpu().numpy()[..., 2 * half:], x[..., 2 * half:])


def _freq(r, base, device):
    return rotary_frequencies(r, base, device=device)[0]


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,hq,hk,d,r", [(1, 32, 8, 128, 128), (5, 14, 2, 64, 64), (37, 28, 4, 128, 64),
                                              (3, 1, 1, 64, 16), (130, 3, 1, 80, 20), (9, 2, 2, 128, 74),
                                              (2, 5, 3, 2, 2), (4100, 2, 1, 64, 32), (7, 1, 1, 512, 512),
                                              (6, 4, 1, 66, 34), (5, 16, 16, 192, 64)])
def test_rotary(cuda, tokens, hq, hk, d, r, dtype, inter):
    g = torch.Generator(device=cuda).manual_seed(tokens * d + r)
    q = torch.randn((tokens, hq, d), generator=g, device=cuda).to(dtype)
    k = torch.randn((tokens, hk, d), generator=g, device=cuda).to(dtype)
    pos = torch.randint(-5, 1 << 20, (tokens,), generator=g, device=cuda)
    freq = _freq(r, 1e4, cuda)
    for inverse, scale in ((False, 1.0), (True, 1.25)):
        qo, ko = apply_rotary(q, k, pos, freq, interleaved=inter, scale=scale, inverse=inverse)
        _check(qo, q, pos, freq, inter, scale, inverse)
        _check(ko, k, pos, freq, inter, scale, inverse)


@pytest.mark.parametrize("offset", [0, 1, 2, 4, 8])
def test_rotary_strided_in_place_and_unaligned(cuda, offset):
    """Rows of a fused projection at any element offset; in place, only the two slices change."""
    g = torch.Generator(device=cuda).manual_seed(offset)
    hq, hk, d, t = 6, 2, 64, 33
    x = torch.randn((t, (hq + 2 * hk) * d + 2 * offset), generator=g, device=cuda).to(torch.bfloat16)
    before = x.clone()
    q = x[:, offset:offset + hq * d].view(t, hq, d) if offset == 0 else x[:, offset:offset + hq * d].unflatten(1, (hq, d))
    k = x[:, offset + hq * d:offset + (hq + hk) * d].unflatten(1, (hk, d))
    q0, k0 = q.clone(), k.clone()
    pos = torch.arange(t, device=cuda) * 1000
    freq = _freq(48, 1e6, cuda)
    fresh = apply_rotary(q, k, pos, freq)
    assert torch.equal(x, before)
    res = apply_rotary(q, k, pos, freq, out=(q, k))
    assert res[0] is q and torch.equal(q, fresh[0]) and torch.equal(k, fresh[1])
    _check(q, q0, pos, freq, False)
    _check(k, k0, pos, freq, False)
    keep = torch.ones_like(x, dtype=torch.bool)
    keep[:, offset:offset + (hq + hk) * d] = False
    assert torch.equal(x[keep], before[keep])


def test_rotary_last_dim_strided_no_k_and_no_tokens(cuda):
    q = torch.randn((4, 64, 3), device=cuda).transpose(1, 2)  # [4, 3, 64], last dim strided
    pos, freq = torch.tensor([3, 1, 1, 0], device=cuda), _freq(64, 1e4, cuda)
    qo, ko = apply_rotary(q, None, pos, freq)
    assert ko is None
    _check(qo, q, pos, freq, False)
    assert torch.equal(qo[3], q[3].contiguous())  # position 0 turns nothing
    e = apply_rotary(q[:0], q[:0], pos[:0], freq)
    assert e[0].shape == (0, 3, 64)


@pytest.mark.parametrize("inter", [False, True])
def test_rotary_copied_dims_keep_what_is_not_finite(cuda, inter):
    q = torch.randn((3, 2, 64), device=cuda).to(torch.bfloat16)
    q[0, 0, 40], q[1, 1, 63], q[2, 0, 33] = float("nan"), float("inf"), -float("inf")
    y, _ = apply_rotary(q, None, torch.arange(3, device=cuda), _freq(32, 1e4, cuda), interleaved=inter)
    assert torch.equal(y[..., 32:].view(torch.int16), q[..., 32:].view(torch.int16))
    assert torch.isfinite(y[..., :32]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inter", [False, True])
def test_rotary_gradient(cuda, dtype, inter):
    """The gradient is the formula's, and (float32) differences agree; broadcast and strided gradients too."""
    g = torch.Generator(device=cuda).manual_seed(3)
    q = torch.randn((11, 6, 64), generator=g, device=cuda).to(dtype).requires_grad_()
    k = torch.randn((11, 2, 64), generator=g, device=cuda).to(dtype).requires_grad_()
    pos, freq = torch.randint(0, 40000, (11,), generator=g, device=cuda), _freq(48, 1e4, cuda)
    gq = torch.randn((11, 6, 64), generator=g, device=cuda).to(dtype)
    gk = torch.randn((1, 1, 64), generator=g, device=cuda).to(dtype).expand(11, 2, 64)
    qo, ko = apply_rotary(q, k, pos, freq, interleaved=inter, scale=1.5)
    got = torch.autograd.grad([qo, ko], [q, k], [gq, gk])
    _check(got[0], gq, pos, freq, inter, 1.5, True)
    _check(got[1], gk, pos, freq, inter, 1.5, True)
    # one of the two alone
    qo, _ = apply_rotary(q, k.detach(), pos, freq, interleaved=inter, scale=1.5)
    assert torch.equal(torch.autograd.grad(qo, q, gq)[0], got[0])
    if dtype == torch.float32:
        e = torch.randn(q.shape, generator=g, device=cuda)
        with torch.no_grad():
            up = apply_rotary(q + 0.5 * e, None, pos, freq, interleaved=inter, scale=1.5)[0]
            down = apply_rotary(q - 0.5 * e, None, pos, freq, interleaved=inter, scale=1.5)[0]
        # linear: the difference is exact but for 24-bit roundings of values below 16, 4,224 of them summed
        torch.testing.assert_close(((up - down).double() * gq.double()).sum(), (got[0].double() * e.double()).sum(),
                                   rtol=0, atol=4224 * 16 * 2.0 ** -22)


def test_rotary_backward_twice_and_captured(cuda):
    """A gradient of the gradient; a forward pass captured and replayed with other positions."""
    q = torch.randn((4, 2, 64), device=cuda, requires_grad=True)
    pos, freq = torch.arange(4, device=cuda), _freq(64, 1e4, cuda)
    y, _ = apply_rotary(q, None, pos, freq)
    (gr,) = torch.autograd.grad(y.square().sum(), q, create_graph=True)
    (g2,) = torch.autograd.grad(gr.sum(), q)
    # |R q|^2 = |q|^2: the gradient is 2 q, its own sum's 2 (a few roundings of values below 8)
    torch.testing.assert_close(gr, 2 * q, rtol=0, atol=2.0 ** -18)
    torch.testing.assert_close(g2, torch.full_like(q, 2.0), rtol=0, atol=2.0 ** -18)
    x = q.detach().clone()
    apply_rotary(x, None, pos, freq)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = apply_rotary(x, None, pos, freq)
    for p in (0, 9, 77):
        pos.copy_(torch.arange(4, device=cuda) + p)
        graph.replay()
        assert torch.equal(out, apply_rotary(x, None, pos, freq)[0])


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("r", [128, 72])
def test_rotary_of_many_rows_is_that_of_few(cuda, r, inter):
    """A batch far larger than the caches gives the bits of its parts turned alone."""
    tokens = 7003
    gen = torch.Generator(device=cuda).manual_seed(r)
    q, k = (torch.randn((tokens, h, 128), generator=gen, device=cuda).to(torch.bfloat16) for h in (32, 8))
    pos = torch.randint(0, 40000, (tokens,), generator=gen, device=cuda)
    freq, scale = rotary_frequencies(r, 1e6, device=cuda)
    gq, gk = apply_rotary(q, k, pos, freq, interleaved=inter, scale=scale)
    for i in range(0, tokens, 1500):
        rows = slice(i, min(i + 1500, tokens))
        wq, wk = apply_rotary(q[rows], k[rows], pos[rows], freq, interleaved=inter, scale=scale)
        assert torch.equal(gq[rows], wq) and torch.equal(gk[rows], wk)


@pytest.mark.parametrize("need_q,need_k,use_q,use_k", [(True, True, True, False), (True, True, False, True),
                                                       (True, False, True, True), (False, True, True, True)])
def test_rotary_gradient_of_one_alone(cuda, need_q, need_k, use_q, use_k):
    """The transpose's rows for what needs a gradient; nothing for a result that is not used."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    q, k = (torch.randn((5, h, 64), generator=gen, device=cuda) for h in (4, 2))
    gq, gk = (torch.randn((5, h, 64), generator=gen, device=cuda) for h in (4, 2))
    pos, (freq, _) = torch.arange(5, device=cuda) * 100, rotary_frequencies(64, device=cuda)
    q.requires_grad_(need_q), k.requires_grad_(need_k)
    yq, yk = apply_rotary(q, k, pos, freq)
    loss = sum((y * g).sum() for y, g, use in ((yq, gq, use_q), (yk, gk, use_k)) if use)
    loss.backward()
    wq, wk = apply_rotary(gq, gk, pos, freq, inverse=True)
    for x, want, got_any in ((q, wq, need_q and use_q), (k, wk, need_k and use_k)):
        if got_any:
            assert torch.equal(x.grad, want)
        else:
            assert x.grad is None or not x.grad.any()


def test_rotary_refusals(cuda):
    q, k = torch.zeros((3, 2, 64), device=cuda), torch.zeros((3, 1, 64), device=cuda)
    pos, freq = torch.arange(3, device=cuda), _freq(64, 1e4, cuda)
    for bad in (dict(q=q.double()), dict(q=q[0]), dict(k=k[:2]), dict(k=k.half()), dict(positions=pos.int()),
                dict(positions=pos[:2]), dict(inv_freq=freq.float()), dict(inv_freq=torch.cat([freq, freq])),
                dict(positions=pos.cpu()), dict(out=(q,)), dict(out=(q, None)), dict(out=(q, k.half())),
                dict(out=(q, k[:1].expand(3, 1, 64))), dict(q=q.clone().requires_grad_(), out=(q, k))):
        args = dict(q=q, k=k, positions=pos, inv_freq=freq)
        args.update(bad)
        with pytest.raises(ValueError):
            apply_rotary(**args)
    with pytest.raises(ValueError, match="head_dim"):
        apply_rotary(torch.zeros((1, 1, 514), device=cuda), None, pos[:1], freq)
