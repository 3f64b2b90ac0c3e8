"""Bounds of the kernels that norm and turn heads against the float64 oracle.

u = 2^-24, half a unit of float32. A rotation (see test_gpu_rotary.py) is off by at most 16 u scale (|a| + |b|).
A norm: a lane sums at most 16 squares and a butterfly of 6 adds the lanes, so the sum (no term is negative) is off
by 23 u of itself, the mean and eps added 25 u; its reciprocal square root by half of that and the function's 2 u:
15 u; with the weight (the offset added: u) and two products 18 u. Together 16 + 18 < 40 u of the size that a
value and its pair's other one have.

The gradient, z = R^T g, m = z w, S = scale (|g_a| + |g_b|) |w|, B = r^2 mean(S |x|): m is off by 18 u S, sum(m x) by
(18 + 24) u sum(S |x|), r^2 by 32 u, so x r^2 mean(m x) by 80 u |x| B, and dx = r (m - ..) by 100 u r (S + |x| B).

A weight's gradient sums z x r, each off by 35 u scale (|g_a| + |g_b|) |x| r: at most 50 of them in a lane of the tests'
sizes, 10 butterflies and waves, 64 workgroups' sums in a row and 16 waves: 35 + 140 < 200 u of the sum of sizes.

A result's own rounding is half a step of its type.
"""

import numpy as np
import torch

from oracle import heads

U = 2.0 ** -24


def f64(x):
    return None if x is None else x.detach().double().cpu().numpy()


def size(x, half, inter, scale):
    """scale (|x_a| + |x_b|) at both of a pair, |x| elsewhere."""
    s = np.abs(x)
    if half:
        a, b = heads.pairs(half, inter)
        s[..., a] = s[..., b] = abs(scale) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return s


def check(got, want, bound, what):
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * np.abs(want) + bound + fi.smallest_normal * fi.eps
    err = np.abs(f64(got) - want)
    assert np.isfinite(f64(got)).all(), what
    assert (err <= tol).all(), f"{what}: off by {(err / tol).max():.3f} of the tolerance"


def check_forward(got, x, w, eps, angle, offset, inter, scale):
    x, w = f64(x), f64(w)
    half = 0 if angle is None else angle.shape[1]
    n = heads.norm(x, w, eps, offset)
    check(got, heads.turn(n, angle, inter, scale), 40 * U * size(n, half, inter, scale), "forward")


def check_backward(dx, dw, x, g, w, eps, angle, offset, inter, scale):
    dt = x.dtype
    x, g, w = f64(x), f64(g), f64(w)
    half = 0 if angle is None else angle.shape[1]
    want, want_w = heads.norm_turn_grad(x, g, w, eps, angle, offset=offset, interleaved=inter, scale=scale)
    r = 1 / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps)
    z = size(g, half, inter, scale)
    s = z if w is None else z * np.abs(w + offset)
    if dx is not None:
        assert dx.dtype == dt
        b = r * r * np.mean(s * np.abs(x), axis=-1, keepdims=True)
        check(dx, want, 100 * U * r * (s + np.abs(x) * b), "dx")
    if dw is not None:
        check(dw, want_w, 200 * U * (z * np.abs(x) * r).sum((0, 1) if w.ndim == 1 else 0), "dw")
