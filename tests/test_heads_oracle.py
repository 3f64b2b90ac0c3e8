"""The oracle of heads normed and turned: against the rotary oracle, and its gradients against differences."""

import numpy as np
import pytest

from oracle import heads, tree


@pytest.mark.parametrize("inter", [False, True])
def test_turn_is_the_rotary_oracle(inter):
    rng = np.random.default_rng(0)
    x, pos, freq = rng.standard_normal((5, 3, 12)), rng.integers(-9, 99, 5), 10.0 ** -np.arange(4)
    want = tree.rotary(x, pos, freq, interleaved=inter, scale=1.5)
    np.testing.assert_allclose(heads.turn(x, heads.phases(pos, freq), inter, 1.5), want, rtol=0, atol=1e-12)
    axes = np.array([0, 2, 1, 7])
    got = heads.phases(np.stack([pos, pos + 1, pos + 2]), freq, axes)
    np.testing.assert_allclose(got, np.stack([pos, pos + 2, pos + 1, 0 * pos], 1) * freq)


@pytest.mark.parametrize("each", [False, True])
def test_gradients_against_differences(each):
    rng = np.random.default_rng(1)
    x, g = rng.standard_normal((4, 2, 10)), rng.standard_normal((4, 2, 10))
    w = rng.standard_normal((2, 10) if each else 10)
    angle = heads.phases(np.arange(4), np.array([1.0, 0.1, 0.3]))
    kw = dict(offset=0.5, interleaved=True, scale=0.7)
    dx, dw = heads.norm_turn_grad(x, g, w, 1e-3, angle, **kw)

    def loss(x, w):
        return (heads.norm_turn(x, w, 1e-3, angle, **kw) * g).sum()

    h = 1e-5
    for a, d in ((x, dx), (w, dw)):
        for at in np.ndindex(*a.shape):
            e = np.zeros_like(a)
            e[at] = h
            diff = (loss(x + e, w) - loss(x - e, w)) if a is x else (loss(x, w + e) - loss(x, w - e))
            assert abs(diff / (2 * h) - d[at]) < 1e-7
