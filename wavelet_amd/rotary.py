"""Rotary positions: queries and keys turned by their tokens' positions before the append and the attention.

The engine applies its model's rotary embedding between the projections and the attention of every
layer (inside ``llm.generate``, wavelet/inference/engine.py:887; the reference patches one model's,
wavelet/inference/deepseek_v4.py:15-126). ``rotary_frequencies`` gives a model's angle per position
for each pair of dims, with the scalings for long contexts in use; ``apply_rotary`` turns ``q`` and
``k`` in one launch, for prompts, single tokens and drafted trees (any positions), and under autograd
for training. Positions may have several axes (time, height and width of images and video):
``rotary_axes`` deals the pairs out to them.
"""

from __future__ import annotations

import ctypes
import math

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib
from .cache import _on, _require_cuda, _stream

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # include/wkv.h, wkv_rotary
MAX_HEAD_DIM = 512  # WKV_ROTARY_MAX_DIM


def _number(scaling: dict, name: str, default=None) -> float:
    v = scaling.get(name, default)
    if v is None:
        raise ValueError(f"rope scaling {_kind(scaling)!r} needs {name!r}")
    return float(v)


def _kind(scaling: dict) -> str:
    return scaling.get("rope_type", scaling.get("type", "default"))


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: dict | None = None,
                       device: torch.device | str | None = None) -> tuple[torch.Tensor, float]:
    """``(inv_freq, scale)`` of a rotary embedding: float64 ``[rotary_dim / 2]`` on ``device`` (default: the
    current GPU), the angle that pair ``i`` gains per position, and the factor of the turned values.

    Without ``scaling`` (and for ``"mrope"``, whose ``mrope_section`` is ``rotary_axes``'s):
    ``base ** (-2 i / rotary_dim)`` and 1. ``scaling`` is a model config's
    ``rope_scaling`` dict, by its ``rope_type``:

    * ``"linear"``: positions divided by ``factor``;
    * ``"dynamic"``: ``base`` raised for a context of ``max_length`` tokens (a key of this dict; at most
      ``original_max_position_embeddings``: not scaled): times ``(factor max_length / original -
      (factor - 1)) ** (rotary_dim / (rotary_dim - 2))``;
    * ``"llama3"``: pairs that turn fewer than ``low_freq_factor`` times over
      ``original_max_position_embeddings`` positions are slowed by ``factor``, those of more than
      ``high_freq_factor`` turns are kept, the ones between interpolated in their number of turns;
    * ``"yarn"``: pairs slowed by ``factor``, kept, or between by a ramp over the pair index from the pair of
      ``beta_fast`` turns (32) to that of ``beta_slow`` (1); values times ``attention_factor``
      (``0.1 ln(factor) + 1``; with ``mscale`` and ``mscale_all_dim``, the ratio of the two such factors).
    """
    rotary_dim = int(rotary_dim)
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even (got {rotary_dim})")
    base = float(base)
    if not base > 0:
        raise ValueError(f"base must be positive (got {base})")
    half = rotary_dim // 2
    scale = 1.0
    kind = "default" if scaling is None else _kind(scaling)
    if kind == "dynamic":
        if rotary_dim == 2:
            raise ValueError("dynamic rope scaling needs more than one pair")
        factor, original = _number(scaling, "factor"), _number(scaling, "original_max_position_embeddings")
        length = max(_number(scaling, "max_length"), original)
        base *= (factor * length / original - (factor - 1)) ** (rotary_dim / (rotary_dim - 2))
    freq = [base ** (-2.0 * i / rotary_dim) for i in range(half)]
    if kind == "linear":
        freq = [f / _number(scaling, "factor") for f in freq]
    elif kind == "llama3":
        factor, original = _number(scaling, "factor"), _number(scaling, "original_max_position_embeddings")
        low, high = _number(scaling, "low_freq_factor"), _number(scaling, "high_freq_factor")
        if not high > low:
            raise ValueError("llama3 rope scaling needs high_freq_factor > low_freq_factor")
        out = []
        for f in freq:
            turns = original * f / (2 * math.pi)
            keep = min(max((turns - low) / (high - low), 0.0), 1.0)
            out.append(keep * f + (1 - keep) * f / factor)
        freq = out
    elif kind == "yarn":
        factor, original = _number(scaling, "factor"), _number(scaling, "original_max_position_embeddings")
        fast, slow = _number(scaling, "beta_fast", 32.0), _number(scaling, "beta_slow", 1.0)

        def pair(turns: float) -> float:  # the (fractional) pair that turns so often over the original context
            return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = pair(fast), pair(slow)
        if scaling.get("truncate", True):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, rotary_dim - 1)
        hi = hi if hi > lo else lo + 0.001
        ramp = [min(max((i - lo) / (hi - lo), 0.0), 1.0) for i in range(half)]
        freq = [f / factor * r + f * (1 - r) for f, r in zip(freq, ramp)]

        def gain(m: float) -> float:
            return 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0

        if scaling.get("attention_factor") is not None:
            scale = float(scaling["attention_factor"])
        elif scaling.get("mscale") and scaling.get("mscale_all_dim"):
            scale = gain(float(scaling["mscale"])) / gain(float(scaling["mscale_all_dim"]))
        else:
            scale = gain(1.0)
    elif kind not in ("default", "dynamic", "mrope"):
        raise NotImplementedError(f"rope scaling {kind!r} is not supported (linear, dynamic, llama3, yarn, mrope)")
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    return torch.tensor(freq, dtype=torch.float64, device=dev), scale


def rotary_axes(sections, *, interleaved: bool = False, device: torch.device | str | None = None) -> torch.Tensor:
    """The axis of every pair (int32 ``[sum(sections)]`` on ``device``, default: the current GPU) where axis ``a``
    of the positions turns ``sections[a]`` pairs of a head.

    The axes' pairs follow each other (a model config's ``mrope_section``), or are dealt out in turn if
    ``interleaved`` (``mrope_interleaved``): axis ``a > 0`` gets pairs ``a``, ``a + n``, ... of ``n`` axes, as many as its
    section says, and axis 0 the others.
    """
    sections = [int(s) for s in sections]
    if not sections or min(sections) < 0 or sum(sections) == 0:
        raise ValueError(f"sections must be non-negative counts of pairs, one an axis (got {sections})")
    n, half = len(sections), sum(sections)
    axes = [a for a, s in enumerate(sections) for _ in range(s)]
    if interleaved:
        axes = [0] * half
        for a, s in enumerate(sections[1:], 1):
            if s > 0 and a + n * (s - 1) >= half:
                raise ValueError(f"sections {sections} cannot take turns over {half} pairs")
            axes[a:a + n * s:n] = [a] * s
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    return torch.tensor(axes, dtype=torch.int32, device=dev)


def check_rotation(positions, inv_freq, axes, tokens: int, d: int, dev: torch.device):
    """A call's positions, frequencies and axes (None: one), checked and contiguous."""
    _require_cuda(positions, "positions", dev)
    shape = positions.shape
    if axes is None:
        if positions.dtype is not torch.int64 or len(shape) != 1 or shape[0] != tokens:
            raise ValueError(f"positions must be int64 [{tokens}] (got {positions.dtype} {tuple(shape)})")
    elif positions.dtype is not torch.int64 or len(shape) != 2 or not shape[0] or shape[1] != tokens:
        raise ValueError(f"positions must be int64 [axes, {tokens}] (got {positions.dtype} {tuple(shape)})")
    _require_cuda(inv_freq, "inv_freq", dev)
    if inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 or not 0 < 2 * inv_freq.shape[0] <= d:
        raise ValueError(f"inv_freq must be float64 [R / 2] with R <= {d} (got {inv_freq.dtype} {tuple(inv_freq.shape)})")
    if axes is not None:
        _require_cuda(axes, "axes", dev)
        if axes.dtype is not torch.int32 or axes.shape != inv_freq.shape:
            raise ValueError(f"axes must be int32 {list(inv_freq.shape)}, one a pair (got {axes.dtype} {tuple(axes.shape)})")
        axes = axes.contiguous()
    return positions.contiguous(), inv_freq.contiguous(), axes


def rotation(positions, inv_freq, axes, interleaved: bool, scale: float, inverse: bool = False) -> _lib.WkvRotary:
    """The library's description of a rotation (wkv_rotary_t) from checked tensors, which have to outlive it."""
    r = 2 * inv_freq.shape[0]
    if axes is None:
        return _lib.WkvRotary(positions.data_ptr(), 0, None, inv_freq.data_ptr(), 1, r, interleaved, inverse, scale, 0)
    return _lib.WkvRotary(positions.data_ptr(), positions.stride(0), axes.data_ptr(), inv_freq.data_ptr(),
                          positions.shape[0], r, interleaved, inverse, scale, 0)


def _launch(q, k, positions, inv_freq, axes, interleaved: bool, scale: float, inverse: bool, out):
    """One launch over checked tensors (k and axes may be None)."""
    qi = q if q.stride(2) == 1 else q.contiguous()
    qo = torch.empty_like(qi, memory_format=torch.contiguous_format) if out is None else out[0]
    tokens, hq, d = qi.shape
    st, sh, _ = qi.stride()
    ot, oh, _ = qo.stride()
    ko = None
    if k is None:
        tail = (None, 0, 0, None, 0, 0, 0)
    else:
        ki = k if k.stride(2) == 1 else k.contiguous()
        ko = torch.empty_like(ki, memory_format=torch.contiguous_format) if out is None else out[1]
        tail = (ki.data_ptr(), *ki.stride()[:2], ko.data_ptr(), *ko.stride()[:2], ki.shape[1])
    dev = q.device
    rows = (_DTYPES[q.dtype], qi.data_ptr(), st, sh, qo.data_ptr(), ot, oh, hq, *tail, d)
    with _on(dev):
        if axes is None:
            rc = _lib.load().wkv_rotary(*rows, positions.data_ptr(), inv_freq.data_ptr(), 2 * inv_freq.shape[0],
                                        interleaved, inverse, scale, tokens, _stream(dev))
        else:
            how = rotation(positions, inv_freq, axes, interleaved, scale, inverse)
            rc = _lib.load().wkv_rotary_axes(*rows, ctypes.byref(how), tokens, _stream(dev))
    _lib.check(rc, "apply_rotary")
    return qo, ko


def _dual(*tensors) -> bool:
    """Whether any of them carries a tangent (forward-mode derivatives)."""
    return _forward_ad._current_level >= 0 and any(
        t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _Rotary(torch.autograd.Function):
    """The rotation is linear and its transpose turns the other way: the backward pass is the same launch
    with the angles negated (and differentiable again), a tangent's the launch itself."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, axes, interleaved, scale, inverse):
        ctx.save_for_backward(positions, inv_freq, axes)
        ctx.save_for_forward(positions, inv_freq, axes)
        ctx.how = (interleaved, scale, inverse)
        ctx.heads = (q.shape[1], None if k is None else k.shape[1])
        ctx.set_materialize_grads(False)
        return _launch(q, k, positions, inv_freq, axes, interleaved, scale, inverse, None)

    @staticmethod
    def backward(ctx, gq, gk):
        gq, gk = (g if need else None for g, need in zip((gq, gk), ctx.needs_input_grad))
        lone = gk if gq is None else None  # k's alone
        if gq is not None or gk is not None:
            interleaved, scale, inverse = ctx.how
            gq, gk = _turned(gq if lone is None else lone, gk if lone is None else None, *ctx.saved_tensors, interleaved,
                             scale, not inverse)
        if lone is not None:
            gq, gk = None, gq
        return gq, gk, None, None, None, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        some, k_heads = tk if tq is None else tq, ctx.heads[1]
        if tq is None:  # (autograd takes no result without a tangent next to one with)
            tq = some.new_zeros((some.shape[0], ctx.heads[0], some.shape[2]))
        if tk is None and k_heads is not None:
            tk = some.new_zeros((some.shape[0], k_heads, some.shape[2]))
        return _turned(tq, tk, *ctx.saved_tensors, *ctx.how)


def _differentiable(q, k) -> bool:
    """Whether autograd has to know of their rotation."""
    return torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)) or _dual(q, k)


def _turned(q, k, *how):
    return _Rotary.apply(q, k, *how) if _differentiable(q, k) else _launch(q, k, *how, None)


def apply_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *,
                 axes: torch.Tensor | None = None, interleaved: bool = False, scale: float = 1.0, inverse: bool = False,
                 out: tuple[torch.Tensor, torch.Tensor | None] | None = None):
    """``q [T, Hq, D]`` and ``k [T, Hk, D]`` (or None) with their heads turned by ``positions [T]`` int64 -> new
    tensors ``(q, k)``.

    bf16, fp16 or fp32, both alike; strided rows (a slice of a fused projection) are read in place.
    ``inv_freq`` (float64 ``[R / 2]``, ``R <= D``) and ``scale`` come from ``rotary_frequencies``: pair ``i``
    of a head is turned by ``positions[t] * inv_freq[i]`` and multiplied by ``scale``. A pair is dims ``(i,
    i + R / 2)``, or ``(2 i, 2 i + 1)`` if ``interleaved``; dims from ``R`` on stay as they are. Positions
    may be any, in any order (a drafted tree's depths; far ones keep the angle that float64 gives). ``inverse``
    turns back (the transpose, also by ``scale``). With ``axes`` (int32 ``[R / 2]``, from ``rotary_axes``) the
    positions are int64 ``[A, T]`` and pair ``i`` is turned by those of axis ``axes[i]`` (a pair of an axis outside
    ``[0, A)`` by none). ``out``: the two results' tensors; ``out=(q, k)`` works in
    place, other tensors share no memory with ``q`` and ``k``. Differentiable in ``q`` and ``k``, forward
    mode too (not with ``out``). For an MLA layer, ``q_pe`` and ``k_pe[:, None]``.
    """
    if not isinstance(q, torch.Tensor) or q.dim() != 3 or q.dtype not in _DTYPES:
        raise ValueError("q must be a bfloat16, float16 or float32 [T, Hq, D] tensor")
    dev = q.device
    if dev.type != "cuda":
        raise ValueError(f"q is on {dev}: apply_rotary runs on the GPU")
    tokens, _, d = q.shape
    if k is not None and (not isinstance(k, torch.Tensor) or k.dim() != 3 or k.dtype != q.dtype or k.device != dev
                          or k.shape[0] != tokens or k.shape[2] != d):
        raise ValueError(f"k must be {q.dtype} [{tokens}, Hk, {d}] on {dev}")
    how = (*check_rotation(positions, inv_freq, axes, tokens, d, dev), bool(interleaved), float(scale), bool(inverse))
    if out is None:
        return _turned(q, k, *how)
    if len(out) != 2 or (out[1] is None) != (k is None):
        raise ValueError("out must hold the results' two tensors (None for no k)")
    written = [o for o in out if o is not None]
    if _differentiable(q, k) or torch.is_grad_enabled() and any(o.requires_grad for o in written) or _dual(*written):
        raise ValueError("out and gradients do not go together: detach q, k and out, or leave out")
    for name, o, x in (("q", out[0], q), ("k", out[1], k)):
        if o is not None and (o.dtype != x.dtype or o.shape != x.shape or o.device != dev or o.stride(2) != 1
                              or (o.shape[0] > 1 and o.stride(0) == 0) or (o.shape[1] > 1 and o.stride(1) == 0)):
            raise ValueError(f"out for {name} must be {x.dtype} {tuple(x.shape)} on {dev} with its last dim contiguous "
                             "and no row twice")
    result = _launch(q, k, *how, out)
    torch.autograd.graph.increment_version(written)  # what autograd saved of them is stale
    return result
