"""Heads normed and turned in one pass, forward and backward, against the float64 oracle (bounds: headcase.py)."""

import numpy as np
import pytest
import torch
from headcase import check_backward, check_forward, f64

from oracle import heads
from wavelet_amd import apply_rotary, norm_rotary, rotary_axes, rotary_frequencies

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
# tokens, query heads, key heads, head dim, turned dims (0: none)
SHAPES = [(1, 32, 8, 128, 128), (5, 14, 2, 64, 64), (37, 28, 4, 128, 64), (3, 1, 1, 64, 16), (130, 3, 1, 80, 20),
          (9, 2, 2, 128, 74), (2, 5, 3, 2, 2), (1030, 2, 1, 64, 32), (7, 1, 1, 512, 512), (6, 4, 1, 66, 34),
          (5, 16, 16, 192, 64), (3, 2, 1, 510, 510), (4, 7, 3, 96, 0), (2, 3, 1, 256, 256), (3, 257, 129, 64, 64),
          (5001, 33, 3, 64, 64)]


def _case(cuda, tokens, hq, hk, d, r, dtype, weights, wide, seed=0):
    g = torch.Generator(device=cuda).manual_seed(tokens * d + r + seed)

    def normal(*shape, dt=dtype):
        return torch.randn(shape, generator=g, device=cuda).to(dt)

    wdt = torch.float32 if wide else dtype
    x = normal(tokens, hq + hk, d) * torch.exp(normal(1, hq + hk, 1, dt=torch.float32)).to(dtype)
    c = dict(q=x[:, :hq], k=x[:, hq:], gq=normal(tokens, hq, d), gk=normal(tokens, hk, d), qw=None, kw=None,
             pos=torch.randint(-5, 1 << 20, (tokens,), generator=g, device=cuda),
             freq=rotary_frequencies(r, 1e4, device=cuda)[0] if r else None)
    if weights:
        c["qw"] = normal(*((hq, d) if weights == "each" else (d,)), dt=wdt)
        c["kw"] = normal(*((hk, d) if weights == "each" else (d,)), dt=wdt)
    if r == 0:
        c["pos"] = None
    c["angle"] = None if r == 0 else heads.phases(f64(c["pos"]), f64(c["freq"]))
    return c


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(cuda, shape, dtype, inter):
    for weights, wide, offset, scale in (("dim", False, 0.0, 1.0), ("each", True, 1.0, 1.25), (None, False, 0.0, 0.5)):
        c = _case(cuda, *shape, dtype, weights, wide)
        q, k = norm_rotary(c["q"], c["k"], c["pos"], c["freq"], q_weight=c["qw"], k_weight=c["kw"], eps=1e-5,
                           weight_offset=offset, interleaved=inter, scale=scale)
        assert q.dtype == dtype and q.is_contiguous() and q.shape == c["q"].shape and k.shape == c["k"].shape
        check_forward(q, c["q"], c["qw"], 1e-5, c["angle"], offset, inter, scale)
        check_forward(k, c["k"], c["kw"], 1e-5, c["angle"], offset, inter, scale)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(cuda, shape, dtype, inter):
    for weights, wide, offset, scale in (("dim", False, 0.0, 1.0), ("each", True, 1.0, 1.25), (None, False, 0.0, 0.5)):
        c = _case(cuda, *shape, dtype, weights, wide)
        leaves = [x.detach().requires_grad_() for x in (c["q"], c["k"])]
        ws = [x if x is None else x.requires_grad_() for x in (c["qw"], c["kw"])]
        q, k = norm_rotary(*leaves, c["pos"], c["freq"], q_weight=ws[0], k_weight=ws[1], eps=1e-5,
                           weight_offset=offset, interleaved=inter, scale=scale)
        wanted = leaves + [w for w in ws if w is not None]
        grads = torch.autograd.grad([q, k], wanted, [c["gq"], c["gk"]], retain_graph=True)
        again = torch.autograd.grad([q, k], wanted, [c["gq"], c["gk"]])
        for a, b in zip(grads, again):
            assert torch.equal(a, b)  # (sums in one order)
        dq, dk, dqw, dkw = (*grads, None, None)[:4]
        check_backward(dq, dqw, c["q"], c["gq"], c["qw"], 1e-5, c["angle"], offset, inter, scale)
        check_backward(dk, dkw, c["k"], c["gk"], c["kw"], 1e-5, c["angle"], offset, inter, scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1401, 66, 8, 64, 64), (3, 64, 1, 64, 64), (1, 33, 2, 128, 32), (1500, 8, 32, 128, 128),
                                   (1100, 17, 2, 512, 64)])
def test_backward_of_long_rows_of_heads(cuda, shape, dtype):
    """Rows of 4,096 elements and more, with one weight, with each head's, and with one of each."""
    c, each = (_case(cuda, *shape, dtype, w, True) for w in ("dim", "each"))
    for qw, kw in ((c["qw"], c["kw"]), (each["qw"], each["kw"]), (c["qw"], each["kw"]), (each["qw"], None)):
        leaves = [x.detach().requires_grad_() for x in (c["q"], c["k"])]
        ws = [None if x is None else x.detach().requires_grad_() for x in (qw, kw)]
        q, k = norm_rotary(*leaves, c["pos"], c["freq"], q_weight=ws[0], k_weight=ws[1], eps=1e-5)
        dq, dk, dqw, dkw = (*torch.autograd.grad([q, k], leaves + [w for w in ws if w is not None], [c["gq"], c["gk"]]),
                            None)[:4]
        check_backward(dq, dqw, c["q"], c["gq"], qw, 1e-5, c["angle"], 0.0, False, 1.0)
        check_backward(dk, dkw, c["k"], c["gk"], kw, 1e-5, c["angle"], 0.0, False, 1.0)


def test_gradients_against_differences(cuda):
    """Derivatives along random directions, by central differences of the float64 oracle: off by h^2 / 6 of a third
    derivative (some 1e-9 here) and the kernel's own bound, a few u of sums of some 4,000 terms of either sign."""
    c = _case(cuda, 9, 3, 1, 96, 64, torch.float32, "dim", False)
    leaves = [x.detach().requires_grad_() for x in (c["q"], c["qw"])]
    q, _ = norm_rotary(leaves[0], None, c["pos"], c["freq"], q_weight=leaves[1], eps=1e-3, scale=1.5)
    dq, dw = torch.autograd.grad(q, leaves, c["gq"])
    x, w, g = f64(c["q"]), f64(c["qw"]), f64(c["gq"])
    rng = np.random.default_rng(5)

    def loss(x, w):
        return (heads.norm_turn(x, w, 1e-3, c["angle"], scale=1.5) * g).sum()

    h = 1e-4
    for _ in range(4):
        vx, vw = rng.standard_normal(x.shape), rng.standard_normal(w.shape)
        got = (f64(dq) * vx).sum()
        size = (np.abs(f64(dq)) * np.abs(vx)).sum()
        assert abs(got - (loss(x + h * vx, w) - loss(x - h * vx, w)) / (2 * h)) < 1e-5 * size
        got, size = (f64(dw) * vw).sum(), (np.abs(f64(dw)) * np.abs(vw)).sum()
        assert abs(got - (loss(x, w + h * vw) - loss(x, w - h * vw)) / (2 * h)) < 1e-5 * size


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("sections,taking_turns", [((16, 24, 24), False), ((24, 20, 20), True), ((32, 32), True),
                                                   ((0, 10, 22), False), ((8,), False)])
def test_axes(cuda, sections, taking_turns, inter):
    d, half = 128, sum(sections)
    axes = rotary_axes(sections, interleaved=taking_turns, device=cuda)
    assert [int((axes == a).sum()) for a in range(len(sections))] == list(sections)
    for dtype in TYPES:
        c = _case(cuda, 29, 5, 2, d, 2 * half, dtype, "dim", False)
        pos = torch.stack([torch.roll(c["pos"], a) + 3 * a for a in range(len(sections))])
        angle = heads.phases(f64(pos), f64(c["freq"]), axes.cpu().numpy())
        leaves = [x.detach().requires_grad_() for x in (c["q"], c["k"], c["qw"], c["kw"])]
        q, k = norm_rotary(leaves[0], leaves[1], pos, c["freq"], q_weight=leaves[2], k_weight=leaves[3], axes=axes,
                           interleaved=inter)
        check_forward(q, c["q"], c["qw"], 1e-6, angle, 0.0, inter, 1.0)
        check_forward(k, c["k"], c["kw"], 1e-6, angle, 0.0, inter, 1.0)
        dq, dk, dqw, dkw = torch.autograd.grad([q, k], leaves, [c["gq"], c["gk"]])
        check_backward(dq, dqw, c["q"], c["gq"], c["qw"], 1e-6, angle, 0.0, inter, 1.0)
        check_backward(dk, dkw, c["k"], c["gk"], c["kw"], 1e-6, angle, 0.0, inter, 1.0)


def test_axis_that_is_not_there(cuda):
    """Its pairs are not turned."""
    c = _case(cuda, 11, 2, 1, 64, 64, torch.float32, "dim", False)
    axes = torch.tensor([0, 1, -1, 2, 1 << 30, -(1 << 31)] + [1] * 26, dtype=torch.int32, device=cuda)
    pos = torch.stack([c["pos"], c["pos"] + 7])
    angle = heads.phases(f64(pos), f64(c["freq"]), axes.cpu().numpy())
    assert (angle[:, 2:6] == 0).all()
    q, _ = norm_rotary(c["q"], None, pos, c["freq"], q_weight=c["qw"], axes=axes)
    check_forward(q, c["q"], c["qw"], 1e-6, angle, 0.0, False, 1.0)
    q, k = apply_rotary(c["q"], c["k"], pos, c["freq"], axes=axes)
    np.testing.assert_array_equal(f64(q)[..., 2:6], f64(c["q"])[..., 2:6])


@pytest.mark.parametrize("offset", [0, 1, 2, 4, 8])
def test_strided_unaligned_and_in_place(cuda, offset):
    c = _case(cuda, 13, 4, 2, 64, 64, torch.bfloat16, "dim", False)
    fused = torch.randn((13, 8 * 64 + offset + 8), device=cuda).bfloat16()
    keep = fused.clone()
    q = fused[:, offset:offset + 4 * 64].view(13, 4, 64)
    k = fused[:, offset + 4 * 64:offset + 6 * 64].view(13, 2, 64)
    want_q, want_k = norm_rotary(q, k, c["pos"], c["freq"], q_weight=c["qw"], k_weight=c["kw"])
    check_forward(want_q, q, c["qw"], 1e-6, c["angle"], 0.0, False, 1.0)
    assert torch.equal(fused, keep)
    gq, gk = norm_rotary(q, k, c["pos"], c["freq"], q_weight=c["qw"], k_weight=c["kw"], out=(q, k))
    assert gq.data_ptr() == q.data_ptr() and torch.equal(q, want_q) and torch.equal(k, want_k)
    rest = torch.ones_like(fused, dtype=torch.bool)
    rest[:, offset:offset + 6 * 64] = False
    assert torch.equal(fused[rest], keep[rest])
    # rows whose heads do not follow each other, and a last dim that is strided
    t = torch.randn((64, 13, 4), device=cuda).bfloat16().permute(1, 2, 0)
    got, _ = norm_rotary(t, None, c["pos"], c["freq"], q_weight=c["qw"])
    check_forward(got, t, c["qw"], 1e-6, c["angle"], 0.0, False, 1.0)
    # weights that start off a 16-byte boundary, and each head's with a row stride of its own
    w = torch.randn((4, 64 + 8 + offset), device=cuda).bfloat16()[:, offset:offset + 64]
    got, _ = norm_rotary(t.contiguous(), None, c["pos"], c["freq"], q_weight=w)
    check_forward(got, t, w, 1e-6, c["angle"], 0.0, False, 1.0)


def test_expanded_gradients_and_heads(cuda):
    """The gradient of a sum, and one head's queries expanded over heads: strides of zero."""
    c = _case(cuda, 21, 1, 1, 64, 64, torch.float32, "dim", False)
    q1 = c["q"].detach().clone().requires_grad_()
    w = c["qw"].detach().requires_grad_()
    q, _ = norm_rotary(q1.expand(21, 6, 64), None, c["pos"], c["freq"], q_weight=w)
    dq, dw = torch.autograd.grad(q.sum(), [q1, w])
    x = q1.detach().expand(21, 6, 64)
    want, want_w = heads.norm_turn_grad(f64(x), np.ones(x.shape), f64(w), 1e-6, c["angle"])
    # 6 heads' gradients of one size added: a few u more than check_backward's
    np.testing.assert_allclose(f64(dq), want.sum(1, keepdims=True), rtol=0, atol=1e-4)
    np.testing.assert_allclose(f64(dw), want_w, rtol=0, atol=1e-3)


@pytest.mark.parametrize("hq", [1, 5, 40])
@pytest.mark.parametrize("dtype", TYPES)
def test_expanded_weights(cuda, dtype, hq):
    """One weight expanded over the heads, each of which has a gradient; their sum (a few u more, within the bound's
    slack) is the one weight's. Also one head's with a head stride of zero."""
    c = _case(cuda, 23, hq, 2, 64, 64, dtype, "dim", True)
    one = [c[x].clone().requires_grad_() for x in ("qw", "kw")]
    wide = one[0].expand(hq, 64) if hq > 1 else one[0].as_strided((1, 64), (0, 1)), one[1].expand(2, 64)
    q, k = norm_rotary(c["q"], c["k"], c["pos"], c["freq"], q_weight=wide[0], k_weight=wide[1], eps=1e-5)
    del_me = [torch.full((hq, 64), float("nan"), device=cuda) for _ in range(2)]  # (what a gradient's memory may hold)
    del del_me
    each = torch.autograd.grad([q, k], wide, [c["gq"], c["gk"]], retain_graph=True)
    both = torch.autograd.grad([q, k], one, [c["gq"], c["gk"]])
    for x, g, w, dw, dw1 in zip((c["q"], c["k"]), (c["gq"], c["gk"]), wide, each, both):
        check_backward(None, dw, x, g, w, 1e-5, c["angle"], 0.0, False, 1.0)
        check_backward(None, dw1, x, g, w[0], 1e-5, c["angle"], 0.0, False, 1.0)


def test_only_some_gradients(cuda):
    c = _case(cuda, 10, 4, 2, 64, 64, torch.bfloat16, "dim", True)
    full = [x.detach().requires_grad_() for x in (c["q"], c["k"], c["qw"], c["kw"])]
    q, k = norm_rotary(full[0], full[1], c["pos"], c["freq"], q_weight=full[2], k_weight=full[3])
    want = torch.autograd.grad([q, k], full, [c["gq"], c["gk"]])
    for i, name in enumerate(("q", "k", "qw", "kw")):
        leaves = [x.detach().requires_grad_(j == i) for j, x in enumerate((c["q"], c["k"], c["qw"], c["kw"]))]
        q, k = norm_rotary(leaves[0], leaves[1], c["pos"], c["freq"], q_weight=leaves[2], k_weight=leaves[3])
        got, = torch.autograd.grad([q, k], [leaves[i]], [c["gq"], c["gk"]])
        # (the grid, and with it the order of a weight's sum, follows the kinds of heads that take part)
        assert torch.equal(got, want[i]) if i < 2 else torch.allclose(got, want[i], rtol=1e-4, atol=1e-4), name
    leaves = [x.detach().requires_grad_() for x in (c["q"], c["k"], c["qw"], c["kw"])]
    _, k = norm_rotary(leaves[0], leaves[1], c["pos"], c["freq"], q_weight=leaves[2], k_weight=leaves[3])
    got = torch.autograd.grad([k], leaves, [c["gk"]], allow_unused=True)  # the queries' result is not used
    assert got[0] is None and got[2] is None and torch.equal(got[1], want[1])


def test_once_differentiable_and_no_forward_mode(cuda):
    c = _case(cuda, 3, 2, 1, 64, 64, torch.float32, "dim", False)
    x = c["q"].detach().requires_grad_()
    q, _ = norm_rotary(x, None, c["pos"], c["freq"], q_weight=c["qw"])
    with pytest.raises(NotImplementedError, match="once"):
        torch.autograd.grad(q.square().sum(), x, create_graph=True)
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level(), torch.no_grad():
        dual = fwd.make_dual(c["q"].detach(), torch.ones_like(c["q"]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            norm_rotary(dual, None, c["pos"], c["freq"], q_weight=c["qw"])


def test_no_tokens_and_no_heads(cuda):
    freq = rotary_frequencies(64, 1e4, device=cuda)[0]
    w = torch.ones(64, device=cuda, requires_grad=True)
    for shape, n in (((0, 4, 64), 0), ((3, 0, 64), 3)):
        x = torch.zeros(shape, device=cuda, requires_grad=True)
        q, _ = norm_rotary(x, None, torch.zeros(n, dtype=torch.int64, device=cuda), freq, q_weight=w)
        assert q.shape == shape
        dx, dw = torch.autograd.grad(q, [x, w], torch.zeros_like(q))
        assert dx.shape == shape and (dw == 0).all()


def test_zeros_large_values_and_nan_stay_in_their_head(cuda):
    c = _case(cuda, 4, 3, 1, 128, 128, torch.bfloat16, "dim", False)
    x = c["q"].contiguous().clone()
    clean, _ = norm_rotary(x, None, c["pos"], c["freq"], q_weight=c["qw"])
    x[0, 0] = 0
    x[1, 1, 5] = float("nan")
    x[2, 2, 70] = float("inf")
    got, _ = norm_rotary(x, None, c["pos"], c["freq"], q_weight=c["qw"])
    assert (got[0, 0] == 0).all() and got[1, 1].isnan().any() and got[2, 2].isnan().any()
    same = torch.ones((4, 3), dtype=torch.bool, device=cuda)
    same[0, 0] = same[1, 1] = same[2, 2] = False
    assert torch.equal(got[same], clean[same])
    big = torch.full((1, 1, 128), 2.0 ** 60, device=cuda)  # squares near float32's end
    got, _ = norm_rotary(big, None, eps=1e-6)
    torch.testing.assert_close(got, torch.ones_like(big), rtol=40 * 2.0 ** -24, atol=0)


def test_graph_replays(cuda):
    """Forward and backward captured in one graph, replayed over new inputs with eager work between."""
    c = _case(cuda, 40, 4, 2, 64, 64, torch.bfloat16, "dim", False)
    st = [x.detach().clone().requires_grad_() for x in (c["q"], c["k"], c["qw"], c["kw"])]
    gq, gk = c["gq"].clone(), c["gk"].clone()

    def step(q, k, qw, kw, gq, gk):
        a, b = norm_rotary(q, k, c["pos"], c["freq"], q_weight=qw, k_weight=kw)
        return [a.detach(), b.detach(), *torch.autograd.grad([a, b], [q, k, qw, kw], [gq, gk])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*st, gq, gk)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*st, gq, gk)
    for seed in range(3):
        n = _case(cuda, 40, 4, 2, 64, 64, torch.bfloat16, "dim", False, seed=seed + 1)
        new = [n[x] for x in ("q", "k", "qw", "kw")]
        with torch.no_grad():
            for a, b in zip(st, new):
                a.copy_(b)
        gq.copy_(n["gq"])
        gk.copy_(n["gk"])
        graph.replay()
        torch.cuda.synchronize()
        want = step(*(x.detach().clone().requires_grad_() for x in new), n["gq"], n["gk"])
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_other_stream(cuda):
    c = _case(cuda, 300, 4, 2, 128, 128, torch.bfloat16, "dim", False)
    want = norm_rotary(c["q"], c["k"], c["pos"], c["freq"], q_weight=c["qw"], k_weight=c["kw"])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = norm_rotary(c["q"], c["k"], c["pos"], c["freq"], q_weight=c["qw"], k_weight=c["kw"])
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals(cuda):
    c = _case(cuda, 4, 2, 1, 64, 64, torch.bfloat16, "dim", False)
    ok = dict(q_weight=c["qw"], k_weight=c["kw"])
    args = (c["q"], c["k"], c["pos"], c["freq"])
    for bad in (dict(q_weight=c["qw"][:32]), dict(q_weight=c["qw"].half()), dict(q_weight=c["qw"].cpu()),
                dict(k_weight=torch.ones((3, 64), device=cuda)), dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")),
                dict(eps=1e-50), dict(weight_offset=float("inf")), dict(scale=float("inf")),
                dict(k_weight=c["kw"].float()), dict(axes=torch.zeros(32, dtype=torch.int32, device=cuda)),
                dict(out=(c["q"],)), dict(out=(torch.empty_like(c["q"]), None)),
                dict(out=(torch.empty(2, 4, 64, device=cuda).bfloat16().transpose(0, 1)[..., ::2], c["k"]))):
        with pytest.raises(ValueError):
            norm_rotary(*args, **{**ok, **bad})
    for bad in ((c["q"].double(), c["k"], c["pos"], c["freq"]), (c["q"], c["k"].float(), c["pos"], c["freq"]),
                (c["q"], c["k"], None, c["freq"]), (c["q"], c["k"], c["pos"], None),
                (c["q"], c["k"], c["pos"].int(), c["freq"]), (c["q"], c["k"], c["pos"][:2], c["freq"]),
                (c["q"], None, c["pos"], c["freq"]), (c["q"][..., :63], c["k"][..., :63], c["pos"], c["freq"][:31]),
                (c["q"].cpu(), None, c["pos"], c["freq"])):
        with pytest.raises(ValueError):
            norm_rotary(*bad, **ok)
    x = c["q"].detach().requires_grad_()
    with pytest.raises(ValueError, match="gradients"):
        norm_rotary(x, c["k"], c["pos"], c["freq"], **ok, out=(torch.empty_like(c["q"]), torch.empty_like(c["k"])))
    with pytest.raises(ValueError, match="take turns"):
        rotary_axes((10, 22), interleaved=True, device=cuda)
    with pytest.raises(ValueError):
        rotary_axes((), device=cuda)


def test_two_streams_at_once(cuda):
    """Forward and backward on two streams that nothing orders, over inputs of their own."""
    cs = [_case(cuda, 700, 8, 4, 128, 128, torch.bfloat16, "dim", False, seed=i) for i in range(2)]

    def run(c):
        leaves = [x.detach().requires_grad_() for x in (c["q"], c["k"], c["qw"], c["kw"])]
        q, k = norm_rotary(leaves[0], leaves[1], c["pos"], c["freq"], q_weight=leaves[2], k_weight=leaves[3])
        return [q.detach(), k.detach(), *torch.autograd.grad([q, k], leaves, [c["gq"], c["gk"]])]

    want = [run(c) for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    got = [None, None]
    for _ in range(3):
        for i, (s, c) in enumerate(zip(streams, cs)):
            with torch.cuda.stream(s):
                got[i] = run(c)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_more_than_2_31_elements(cuda):
    """The last tokens of 2^20 + 5 tokens of 16 heads of 128."""
    tokens = (1 << 20) + 5
    freq = rotary_frequencies(128, 1e4, device=cuda)[0]
    q = torch.empty((tokens, 16, 128), dtype=torch.bfloat16, device=cuda).normal_()
    pos = torch.arange(tokens, device=cuda)
    w = torch.ones(128, device=cuda)
    got, _ = norm_rotary(q, None, pos, freq, q_weight=w)
    check_forward(got[-7:], q[-7:], w, 1e-6, heads.phases(f64(pos[-7:]), f64(freq)), 0.0, False, 1.0)
    check_forward(got[:3], q[:3], w, 1e-6, heads.phases(f64(pos[:3]), f64(freq)), 0.0, False, 1.0)
    del got
    leaf = q.detach().requires_grad_()
    out, _ = norm_rotary(leaf, None, pos, freq, q_weight=w)
    dq, = torch.autograd.grad(out, leaf, q)
    check_backward(dq[-5:], None, q[-5:], q[-5:], w, 1e-6, heads.phases(f64(pos[-5:]), f64(freq)), 0.0, False, 1.0)
