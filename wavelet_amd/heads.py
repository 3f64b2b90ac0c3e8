"""Norms of queries and keys for each head, with the rotary positions in the same pass.

Models that norm their heads (a root mean square over each, with weights for queries and keys) do so between
the projections and the rotary embedding of every layer; the engine runs both inside ``llm.generate``
(wavelet/inference/engine.py:887). ``norm_rotary`` reads a head once for the two, in prompts, single tokens
and under autograd for training, with the weights' gradients.
"""

from __future__ import annotations

import torch

from . import _lib
from .cache import _on, _stream
from .rotary import _DTYPES, _dual, check_rotation, rotation


def check_weight(w, name: str, heads: int, x: torch.Tensor):
    """A head norm's weight (None: ones) for ``heads`` heads of ``x``'s type and size, its last dim contiguous."""
    if w is None:
        return None
    if (not isinstance(w, torch.Tensor) or w.device != x.device
            or (w.dtype is not x.dtype and w.dtype is not torch.float32)):
        raise ValueError(f"{name} must be a float32 or {x.dtype} tensor on {x.device}")
    shape, d = w.shape, x.shape[-1]
    if shape != (d,) and shape != (heads, d):
        raise ValueError(f"{name} must be [{d}] or [{heads}, {d}] (got {list(shape)})")
    return w if w.stride(-1) == 1 else w.contiguous()


def head_norm(q_weight, k_weight, eps: float, offset: float) -> _lib.WkvHeadNorm:
    """The library's description of a norm (wkv_head_norm_t) from checked weights, which have to outlive it."""
    qw = kw = None
    qs = ks = dtype = 0
    if q_weight is not None:
        qw, dtype = q_weight.data_ptr(), _DTYPES[q_weight.dtype]
        if q_weight.dim() == 2:
            qs = q_weight.stride(0)
    if k_weight is not None:
        kw = k_weight.data_ptr()
        if q_weight is None:
            dtype = _DTYPES[k_weight.dtype]
        elif k_weight.dtype is not q_weight.dtype:
            raise ValueError(f"q_weight and k_weight must have one type (got {q_weight.dtype} and {k_weight.dtype})")
        if k_weight.dim() == 2:
            ks = k_weight.stride(0)
    return _lib.WkvHeadNorm(qw, kw, qs, ks, dtype, offset, eps, 0)


def _forward(q, k, q_weight, k_weight, rotary, interleaved, scale, eps, offset, out):
    """One launch over checked tensors; rotary: (positions, inv_freq, axes), or None: only normed."""
    tokens, hq, d = q.shape
    dev = q.device
    if q.stride(2) != 1:
        q = q.contiguous()
    if k is not None and k.stride(2) != 1:
        k = k.contiguous()
    if out is None:
        out = (torch.empty_like(q, memory_format=torch.contiguous_format),
               None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format))
    norm = head_norm(q_weight, k_weight, eps, offset)
    how = None if rotary is None else rotation(*rotary, interleaved, scale)  # (a struct goes by reference)
    qo, ko = out
    st, sh, _ = q.stride()
    ot, oh, _ = qo.stride()
    if k is None:
        tail = (None, 0, 0, None, 0, 0, 0)
    else:
        kst, ksh, _ = k.stride()
        kot, koh, _ = ko.stride()
        tail = (k.data_ptr(), kst, ksh, ko.data_ptr(), kot, koh, k.shape[1])
    with _on(dev):
        rc = _lib.load().wkv_norm_rotary(_DTYPES[q.dtype], q.data_ptr(), st, sh, qo.data_ptr(), ot, oh, hq, *tail, d,
                                         norm, how, tokens, _stream(dev))
    if rc:
        _lib.check(rc, "norm_rotary")
    return out


def _grad_rows(x, g, want: bool):
    """A kind's part of the backward call: its result (None: not wanted), and pointers, strides and heads."""
    if x is None:
        return None, (None, 0, 0, None, 0, 0, None, 0, 0, 0)
    xt, xh, last = x.stride()
    if last != 1:
        x = x.contiguous()
        xt, xh, _ = x.stride()
    gt, gh, last = g.stride()
    if last != 1:
        g = g.contiguous()
        gt, gh, _ = g.stride()
    if not want:
        return (None, x, g), (x.data_ptr(), xt, xh, g.data_ptr(), gt, gh, None, 0, 0, x.shape[1])
    d = torch.empty_like(x, memory_format=torch.contiguous_format)
    dt, dh, _ = d.stride()
    return (d, x, g), (x.data_ptr(), xt, xh, g.data_ptr(), gt, gh, d.data_ptr(), dt, dh, x.shape[1])


def _weight_grad(x, w, want: bool):
    """The weight that the launch takes, its gradient, empty, and that one's pointer (None: not wanted; no head, no sum)."""
    if not want or x is None or w is None:
        return w, None, None
    if x.shape[1] == 0:
        return w, torch.zeros_like(w), None
    if w.dim() == 2 and w.shape[0] > 1 and w.stride(0) == 0:
        w = w.contiguous()  # (an expanded weight has a gradient for every head)
    d = torch.empty_like(w, memory_format=torch.contiguous_format)
    return w, d, d.data_ptr()


def _backward(q, k, gq, gk, q_weight, k_weight, rotary, interleaved, scale, eps, offset, need):
    """The gradients (dq, dk, dq_weight, dk_weight) that ``need`` asks for; gq or gk None: zero."""
    if gq is None:
        q = None
    if gk is None:
        k = None
    some = k if q is None else q
    dev = some.device
    tokens, _, d = some.shape
    keep_q, rows_q = _grad_rows(q, gq, need[0])  # (what was copied lives until the launch)
    keep_k, rows_k = _grad_rows(k, gk, need[1])
    q_weight, dqw, dqw_ptr = _weight_grad(q, q_weight, need[2])
    k_weight, dkw, dkw_ptr = _weight_grad(k, k_weight, need[3])
    norm = head_norm(q_weight, k_weight, eps, offset)
    how = None if rotary is None else rotation(*rotary, interleaved, scale)
    lib = _lib.load()
    ws, size, ws_ptr = None, 0, None
    if dqw_ptr is not None or dkw_ptr is not None:
        size = lib.wkv_norm_rotary_workspace_size(tokens, rows_q[-1], rows_k[-1], d,
                                                  norm.q_weight_stride_h != 0, norm.k_weight_stride_h != 0)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        ws_ptr = ws.data_ptr()
    with _on(dev):
        rc = lib.wkv_norm_rotary_backward(_DTYPES[some.dtype], *rows_q, *rows_k, d, norm, how, dqw_ptr, dkw_ptr, tokens,
                                          ws_ptr, size, _stream(dev))
    if rc:
        _lib.check(rc, "norm_rotary backward")
    return None if q is None else keep_q[0], None if k is None else keep_k[0], dqw, dkw


class _NormRotary(torch.autograd.Function):
    """The inputs are kept, not the normed heads: the backward launch norms them again."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, rotary, interleaved, scale, eps, offset):
        ctx.save_for_backward(q, k, q_weight, k_weight, *(rotary or ()))
        ctx.how = (interleaved, scale, eps, offset)
        ctx.set_materialize_grads(False)
        return _forward(q, k, q_weight, k_weight, rotary, interleaved, scale, eps, offset, None)

    @staticmethod
    def backward(ctx, gq, gk):
        if torch.is_grad_enabled():  # (create_graph: the launch's results would count as constants)
            raise NotImplementedError("norm_rotary is differentiable once: its gradients have no create_graph")
        q, k, q_weight, k_weight, *rotary = ctx.saved_tensors
        need = ctx.needs_input_grad[:4]
        gq, gk = (g if need[i] or need[i + 2] else None for i, g in enumerate((gq, gk)))
        if gq is None and gk is None:
            return (None,) * 9
        grads = _backward(q, k, gq, gk, q_weight, k_weight, tuple(rotary) or None, *ctx.how, need)
        return (*grads, None, None, None, None, None)


def norm_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor | None = None,
                inv_freq: torch.Tensor | None = None, *, q_weight: torch.Tensor | None = None,
                k_weight: torch.Tensor | None = None, eps: float = 1e-6, weight_offset: float = 0.0,
                axes: torch.Tensor | None = None, interleaved: bool = False, scale: float = 1.0,
                out: tuple[torch.Tensor, torch.Tensor | None] | None = None):
    """``q [T, Hq, D]`` and ``k [T, Hk, D]`` (or None) with every head normed and turned -> new tensors ``(q, k)``.

    The norm: ``x / sqrt(mean(x ** 2) + eps) * (weight + weight_offset)`` over each head, weights ``[D]`` for all
    heads or ``[H, D]``, of the heads' type or float32 (None: ones, without the offset). The rotation: ``apply_rotary``'s, from
    ``positions``, ``inv_freq``, ``axes``, ``interleaved`` and ``scale`` (``positions`` and ``inv_freq`` None: the heads
    are only normed). bf16, fp16 or fp32, ``D`` even and at most 512, strided rows read in place; all of it is
    computed in float32 and rounded once. ``out``: the two results' tensors; ``out=(q, k)`` works in place, other
    tensors share no memory with the inputs. Differentiable once, in ``q``, ``k`` and the weights (not with ``out``,
    ``create_graph`` or forward mode).
    """
    if not isinstance(q, torch.Tensor) or q.dim() != 3 or q.dtype not in _DTYPES:
        raise ValueError("q must be a bfloat16, float16 or float32 [T, Hq, D] tensor")
    dev = q.device
    if dev.type != "cuda":
        raise ValueError(f"q is on {dev}: norm_rotary runs on the GPU")
    tokens, hq, d = q.shape
    if k is not None and (not isinstance(k, torch.Tensor) or k.dim() != 3 or k.dtype != q.dtype or k.device != dev
                          or k.shape[0] != tokens or k.shape[2] != d):
        raise ValueError(f"k must be {q.dtype} [{tokens}, Hk, {d}] on {dev}")
    q_weight = check_weight(q_weight, "q_weight", hq, q)
    if k is None and k_weight is not None:
        raise ValueError("k_weight without k")
    k_weight = check_weight(k_weight, "k_weight", 0 if k is None else k.shape[1], q)
    if (positions is None) != (inv_freq is None) or (inv_freq is None and axes is not None):
        raise ValueError("positions and inv_freq go together (both None: the heads are only normed)")
    rotary = None if inv_freq is None else check_rotation(positions, inv_freq, axes, tokens, d, dev)
    how = (rotary, bool(interleaved), float(scale), float(eps), float(weight_offset))
    differentiable = _dual(q, k, q_weight, k_weight) or torch.is_grad_enabled() and (
        q.requires_grad or k is not None and k.requires_grad or q_weight is not None and q_weight.requires_grad
        or k_weight is not None and k_weight.requires_grad)
    if out is None:
        if differentiable:
            return _NormRotary.apply(q, k, q_weight, k_weight, *how)
        return _forward(q, k, q_weight, k_weight, *how, None)
    if len(out) != 2 or (out[1] is None) != (k is None):
        raise ValueError("out must hold the results' two tensors (None for no k)")
    written = [o for o in out if o is not None]
    if differentiable or torch.is_grad_enabled() and any(o.requires_grad for o in written) or _dual(*written):
        raise ValueError("out and gradients do not go together: detach q, k, the weights and out, or leave out")
    for name, o, x in (("q", out[0], q), ("k", out[1], k)):
        if o is not None and (o.dtype != x.dtype or o.shape != x.shape or o.device != dev or o.stride(2) != 1
                              or (o.shape[0] > 1 and o.stride(0) == 0) or (o.shape[1] > 1 and o.stride(1) == 0)):
            raise ValueError(f"out for {name} must be {x.dtype} {tuple(x.shape)} on {dev} with its last dim contiguous "
                             "and no row twice")
    result = _forward(q, k, q_weight, k_weight, *how, tuple(out))
    torch.autograd.graph.increment_version(written)  # what autograd saved of them is stale
    return result
