"""Heads normed and turned, in float64: the norm, rotary positions with several axes, and their gradients."""

from __future__ import annotations

import numpy as np


def phases(positions, inv_freq, axes=None) -> np.ndarray:
    """The angle of every token's pairs ``[T, R / 2]``; positions ``[T]``, or ``[A, T]`` with axes ``[R / 2]``."""
    positions, inv_freq = np.asarray(positions, dtype=np.float64), np.asarray(inv_freq, dtype=np.float64)
    if axes is None:
        return positions[:, None] * inv_freq
    axes = np.asarray(axes)
    there = (axes >= 0) & (axes < len(positions))
    return np.where(there, positions[np.where(there, axes, 0)].T, 0.0) * inv_freq


def pairs(half: int, interleaved: bool):
    i = np.arange(half)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + half)


def turn(x, angle, interleaved=False, scale=1.0) -> np.ndarray:
    """``x [T, H, D]`` with its pairs turned by ``angle [T, R / 2]`` (None: as it is)."""
    y = np.array(x, dtype=np.float64)
    if angle is None:
        return y
    a, b = pairs(angle.shape[1], interleaved)
    c, s = (scale * f(angle)[:, None] for f in (np.cos, np.sin))
    xa, xb = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    return y


def norm(x, weight, eps, offset=0.0) -> np.ndarray:
    x = np.asarray(x, dtype=np.float64)
    w = 1.0 if weight is None else np.asarray(weight, dtype=np.float64) + offset
    return x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps) * w


def norm_turn(x, weight, eps, angle=None, *, offset=0.0, interleaved=False, scale=1.0) -> np.ndarray:
    return turn(norm(x, weight, eps, offset), angle, interleaved, scale)


def norm_turn_grad(x, g, weight, eps, angle=None, *, offset=0.0, interleaved=False, scale=1.0):
    """``(dx, dweight)`` of ``norm_turn`` for the gradient ``g`` of its result (dweight None without a weight)."""
    x = np.asarray(x, dtype=np.float64)
    z = turn(g, None if angle is None else -angle, interleaved, scale)
    r = 1 / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps)
    dw = None
    if weight is not None:
        weight = np.asarray(weight, dtype=np.float64)
        dw = (z * x * r).sum((0, 1) if weight.ndim == 1 else 0)
        z = z * (weight + offset)
    return r * (z - x * r * r * np.mean(z * x, axis=-1, keepdims=True)), dw
