"""Rotary positions with several axes against the float64 oracle (bounds: headcase.py, test_gpu_rotary.py)."""

import pytest
import torch
from headcase import U, check, f64, size

from oracle import heads
from wavelet_amd import apply_rotary, rotary_axes, rotary_frequencies

pytestmark = pytest.mark.gpu


def _inputs(cuda, tokens, hq, hk, d, half, n, dtype):
    g = torch.Generator(device=cuda).manual_seed(tokens + d + n)
    q, k, gq, gk = (torch.randn((tokens, h, d), generator=g, device=cuda).to(dtype) for h in (hq, hk, hq, hk))
    pos = torch.randint(-5, 1 << 20, (n, tokens), generator=g, device=cuda)
    return q, k, gq, gk, pos, rotary_frequencies(2 * half, 1e4, device=cuda)[0]


def _check(got, x, angle, inter, scale):
    half = angle.shape[1]
    check(got, heads.turn(f64(x), angle, inter, scale), 16 * U * size(f64(x), half, inter, scale), "rotary")


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,hq,hk,d,sections,turns", [(1, 28, 4, 128, (16, 24, 24), False),
                                                           (37, 14, 2, 64, (12, 10, 10), True),
                                                           (130, 3, 1, 80, (20, 20), False), (5, 2, 2, 72, (9, 9), True),
                                                           (4100, 2, 1, 64, (8, 8, 8, 8), True), (0, 2, 1, 64, (32,), False)])
def test_axes(cuda, tokens, hq, hk, d, sections, turns, dtype, inter):
    half, n = sum(sections), len(sections)
    q, k, gq, gk, pos, freq = _inputs(cuda, tokens, hq, hk, d, half, n, dtype)
    axes = rotary_axes(sections, interleaved=turns, device=cuda)
    angle = heads.phases(f64(pos), f64(freq), axes.cpu().numpy())
    x, y = q.requires_grad_(), k.requires_grad_()
    a, b = apply_rotary(x, y, pos, freq, axes=axes, interleaved=inter, scale=1.25)
    _check(a, q, angle, inter, 1.25)
    _check(b, k, angle, inter, 1.25)
    dq, dk = torch.autograd.grad([a, b], [x, y], [gq, gk])
    _check(dq, gq, -angle, inter, 1.25)
    _check(dk, gk, -angle, inter, 1.25)
    back, _ = apply_rotary(a.detach(), None, pos, freq, axes=axes, interleaved=inter, scale=1 / 1.25, inverse=True)
    _check(back, a, -angle, inter, 1 / 1.25)


def test_equal_axes_are_one(cuda):
    q, k, _, _, pos, freq = _inputs(cuda, 50, 4, 2, 128, 64, 3, torch.bfloat16)
    pos = pos[:1].expand(3, -1)
    want = apply_rotary(q, k, pos[0], freq)
    got = apply_rotary(q, k, pos, freq, axes=rotary_axes((16, 24, 24), device=cuda))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    strided = torch.empty((50, 5), dtype=torch.int64, device=cuda)[:, 1:4].T  # positions whose rows are not contiguous
    strided.copy_(pos)
    got = apply_rotary(q, k, strided, freq, axes=rotary_axes((16, 24, 24), device=cuda))
    assert torch.equal(got[0], want[0])
    x, y = q.clone(), k.clone()
    apply_rotary(x, y, pos, freq, axes=rotary_axes((64,), device=cuda), out=(x, y))
    assert torch.equal(x, want[0]) and torch.equal(y, want[1])


def test_the_axes_of_pairs():
    assert rotary_axes((2, 3, 1), device="cpu").tolist() == [0, 0, 1, 1, 1, 2]
    assert rotary_axes((4, 2, 2), interleaved=True, device="cpu").tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    assert rotary_axes((4, 3, 1), interleaved=True, device="cpu").tolist() == [0, 1, 2, 0, 1, 0, 0, 1]
    freq, scale = rotary_frequencies(16, 1e4, scaling=dict(type="mrope", mrope_section=[2, 3, 3]), device="cpu")
    assert scale == 1.0 and torch.equal(freq, rotary_frequencies(16, 1e4, device="cpu")[0])


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,hq,hk,d,half,shift", [(37, 8, 2, 128, 64, 0), (5, 3, 1, 64, 10, 0), (130, 4, 2, 80, 13, 0),
                                                       (300, 2, 0, 64, 32, 1), (4, 1, 3, 512, 255, 2)])
def test_turn_heads(cuda, tokens, hq, hk, d, half, shift, dtype, inter):
    """wkv_turn_heads, new rows and in place, and the inverse: the rotation of an append without a norm."""
    from wavelet_amd import _lib
    from wavelet_amd.rotary import rotation

    lib = _lib.load()
    _, _, _, _, pos, freq = _inputs(cuda, tokens, 1, 1, d, half, 3, dtype)
    axes = (torch.arange(half, device=cuda) % 3).int()
    x = torch.randn(tokens * (hq + hk) * d + shift, device=cuda).to(dtype)[shift:].view(tokens, hq + hk, d)
    y, angle = torch.full_like(x, float("nan")), heads.phases(f64(pos), f64(freq), axes.cpu().numpy())

    def rows(a, b):
        args = []
        for lo, n in ((0, hq), (hq, hk)):
            for t in (a, b):
                args += [t[:, lo:].data_ptr() if n else None, t.stride(0), t.stride(1)]
            args.append(n)
        return args

    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    stream = torch.cuda.current_stream().cuda_stream
    for way in (False, True):
        how = rotation(pos, freq, axes, inter, 1.25, way)
        _lib.check(lib.wkv_turn_heads(code, *rows(x, y), d, how, tokens, stream), "turn")
        _check(y, x, -angle if way else angle, inter, 1.25)
        z = x.clone()
        _lib.check(lib.wkv_turn_heads(code, *rows(z, z), d, how, tokens, stream), "turn in place")
        _check(z, x, -angle if way else angle, inter, 1.25)
        # (fp16 at another alignment: a fused product and conversion rounds some values once, others twice)
        assert dtype is torch.float16 or torch.equal(y, z)


def test_refusals(cuda):
    q, k, _, _, pos, freq = _inputs(cuda, 6, 2, 1, 64, 32, 3, torch.bfloat16)
    axes = rotary_axes((12, 10, 10), device=cuda)
    for bad in (dict(axes=axes[:31]), dict(axes=axes.long()), dict(axes=axes.cpu()), dict(axes=None)):
        with pytest.raises(ValueError):
            apply_rotary(q, k, pos, freq, **bad)
    for bad in (pos[:, :5], pos.int(), pos[0], pos[:0]):
        with pytest.raises(ValueError):
            apply_rotary(q, k, bad, freq, axes=axes)
    with pytest.raises(ValueError):
        rotary_axes((4, -1), device=cuda)
