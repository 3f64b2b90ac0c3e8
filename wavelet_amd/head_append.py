"""The append with the norm of heads and the rotary positions on the way: what a layer does between its projections
and its attention, in one launch.

The engine norms (where its model does) and turns queries and keys and then appends keys and values to its paged
cache, for every layer of every step inside ``llm.generate`` (wavelet/inference/engine.py:887; the reference's
own sequence is at wavelet/kernels/patch.py:173-196). ``rotary_append`` reads the projections once and writes the
queries for the attention and the cache; ``mla_rotary_append`` is the same for a latent cache.
"""

from __future__ import annotations

import torch

from . import _lib
from .cache import MLALatentCache, PagedKVCache, _on, _require_cuda, _slots, _stream, _token_rows
from .heads import check_weight, head_norm
from .rotary import _dual, check_rotation, rotation


def _no_gradients(what: str, *tensors) -> None:
    """A cache keeps no graph: what goes into it cannot be differentiated."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                break
        else:
            if not _dual(*tensors):
                return
    elif not _dual(*tensors):
        return
    raise ValueError(f"{what} has no gradient: detach its inputs, or call it under torch.no_grad()")


def _result(x: torch.Tensor, out, name: str) -> torch.Tensor:
    """The queries' result: ``out``, checked, or a new tensor."""
    if out is None:
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    if (not isinstance(out, torch.Tensor) or out.dtype != x.dtype or out.shape != x.shape or out.device != x.device
            or out.stride(2) != 1 or (out.shape[0] > 1 and out.stride(0) == 0)
            or (out.shape[1] > 1 and out.stride(1) == 0)):
        raise ValueError(f"out must be {x.dtype} {tuple(x.shape)} on {x.device} for {name}, with its last dim "
                         "contiguous and no row twice")
    return out


def _rows(q, result) -> tuple:
    """Pointers, strides and heads of the queries and their result (None: there are none)."""
    if q is None:
        return None, 0, 0, None, 0, 0, 0
    st, sh, _ = q.stride()
    ot, oh, _ = result.stride()
    return q.data_ptr(), st, sh, result.data_ptr(), ot, oh, q.shape[1]


def _queries(q, name: str, tokens: int, d: int, dev: torch.device) -> torch.Tensor:
    _require_cuda(q, name, dev)
    if q.dtype != torch.bfloat16 or q.dim() != 3 or q.shape[0] != tokens or q.shape[2] != d:
        raise ValueError(f"{name} must be bfloat16 [{tokens}, H, {d}] (got {q.dtype} {tuple(q.shape)})")
    return q if q.stride(2) == 1 else q.contiguous()


def rotary_append(q: torch.Tensor | None, key: torch.Tensor, value: torch.Tensor, cache: PagedKVCache,
                  slot_mapping: torch.Tensor, positions: torch.Tensor | None = None,
                  inv_freq: torch.Tensor | None = None, *, q_weight: torch.Tensor | None = None,
                  k_weight: torch.Tensor | None = None, eps: float | None = None, weight_offset: float = 0.0,
                  axes: torch.Tensor | None = None, interleaved: bool = False, scale: float = 1.0,
                  out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Queries normed and turned -> a new tensor (or ``out``: ``q`` itself, or one that shares no memory with the inputs),
    keys normed and turned and values into ``cache`` at ``slot_mapping`` (-1: skipped).

    ``q [T, Hq, D]`` (None: keys and values only), ``key`` and ``value`` ``[T, Hkv, D]`` bf16, strided rows of a fused
    projection read in place. The norm is ``norm_rotary``'s and is done where ``eps`` is given, the rotation
    ``apply_rotary``'s and done where ``positions`` and ``inv_freq`` are; one of them at least. The attention then
    takes the result and no ``key`` / ``value`` (``paged_decode_gqa``, ``prefill_gqa``, ``paged_tree_gqa``). ``key`` and
    ``value`` are left as they are, and the cache, bf16 or fp8, holds what ``norm_rotary`` and ``cache.append`` would
    leave in it, bit for bit where the key's rows start on 16-byte boundaries (elsewhere they are copied, and then, as
    where ``apply_rotary`` goes first, a key's last bit may differ). A slot appears once in a call, a block of an fp8
    cache in one run of it (as for ``cache.append``). Long prompts into an fp8 cache (16,384 tokens of 8 key heads, or
    blocks of 256) take less time as ``norm_rotary`` and ``cache.append``.
    """
    if not isinstance(cache, PagedKVCache):
        raise ValueError("cache must be a PagedKVCache (mla_rotary_append appends to latent caches)")
    dev, d = cache.device, cache.head_dim
    shape = (cache.num_kv_heads, d)
    key = _token_rows(key, "key", shape, dev)
    value = _token_rows(value, "value", shape, dev)
    tokens = key.shape[0]
    if value.shape[0] != tokens:
        raise ValueError("key and value must have the same number of tokens")
    slots = _slots(slot_mapping, tokens, dev)
    if q is None:
        if out is not None or q_weight is not None:
            raise ValueError("out and q_weight go with q")
    else:
        q = _queries(q, "q", tokens, d, dev)
    if eps is None and (q_weight is not None or k_weight is not None or weight_offset != 0.0):
        raise ValueError("the norm's weights need its eps")
    if (positions is None) != (inv_freq is None) or (inv_freq is None and (axes is not None or eps is None)):
        raise ValueError("a rotation (positions and inv_freq) or a norm (eps) must be given")
    norm = None
    if eps is not None:
        q_weight = None if q is None else check_weight(q_weight, "q_weight", q.shape[1], q)
        k_weight = check_weight(k_weight, "k_weight", shape[0], key)
        norm = head_norm(q_weight, k_weight, float(eps), float(weight_offset))
    how = None
    if inv_freq is not None:
        positions, inv_freq, axes = check_rotation(positions, inv_freq, axes, tokens, d, dev)
        how = rotation(positions, inv_freq, axes, bool(interleaved), float(scale))
    result = None if q is None else _result(q, out, "q")
    _no_gradients("rotary_append", q, key, value, q_weight, k_weight, out)
    kst, ksh, _ = key.stride()
    vst, vsh, _ = value.stride()
    with _on(dev):
        rc = _lib.load().wkv_rotary_append(cache.descriptor(), key.data_ptr(), kst, ksh, value.data_ptr(), vst, vsh,
                                           slots.data_ptr(), *_rows(q, result), norm, how, tokens, _stream(dev))
    if rc:
        _lib.check(rc, "rotary_append")
    if out is not None:
        torch.autograd.graph.increment_version([out])
    return result


def mla_rotary_append(q_pe: torch.Tensor | None, kv_c: torch.Tensor, k_pe: torch.Tensor, cache: MLALatentCache,
                      slot_mapping: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *,
                      kv_weight: torch.Tensor | None = None, eps: float | None = None, weight_offset: float = 0.0,
                      axes: torch.Tensor | None = None, interleaved: bool = False, scale: float = 1.0,
                      out: torch.Tensor | None = None) -> torch.Tensor | None:
    """The queries' ``q_pe [T, H, rope_dim]`` (None: none) turned -> a new tensor (or ``out``, as for ``rotary_append``), and into the latent
    ``cache`` at ``slot_mapping`` (-1: skipped) the compressed entries ``kv_c [T, kv_lora_rank]``, normed where ``eps``
    is given (weight ``[kv_lora_rank]``, None: ones), and ``k_pe [T, rope_dim]`` turned.

    bf16; the rotation as for ``apply_rotary``, the norm as ``norm_rotary``'s over a whole entry. The attention
    (``paged_decode_mla``) then takes the result as its ``q_pe`` and no ``kv_c`` / ``k_pe``. A slot appears once in a call.
    A ``rope_dim`` above 128 needs rows of queries (and, unless ``interleaved``, pairs) in multiples of 2 elements, one
    above 256 (itself a multiple of 16) in multiples of 8; others are refused.
    """
    if not isinstance(cache, MLALatentCache):
        raise ValueError("cache must be an MLALatentCache (rotary_append appends to key and value caches)")
    dev = cache.device
    kv_c = _token_rows(kv_c, "kv_c", (cache.kv_lora_rank,), dev)
    k_pe = _token_rows(k_pe, "k_pe", (cache.rope_dim,), dev)
    tokens = kv_c.shape[0]
    if k_pe.shape[0] != tokens:
        raise ValueError("kv_c and k_pe must have the same number of tokens")
    slots = _slots(slot_mapping, tokens, dev)
    if q_pe is None:
        if out is not None:
            raise ValueError("out goes with q_pe")
    else:
        q_pe = _queries(q_pe, "q_pe", tokens, cache.rope_dim, dev)
    positions, inv_freq, axes = check_rotation(positions, inv_freq, axes, tokens, cache.rope_dim, dev)
    how = rotation(positions, inv_freq, axes, bool(interleaved), float(scale))
    norm = None
    if eps is None:
        if kv_weight is not None or weight_offset != 0.0:
            raise ValueError("the norm's weight needs its eps")
    else:
        if kv_weight is not None:
            kv_weight = check_weight(kv_weight, "kv_weight", 1, kv_c)
            if kv_weight.dim() != 1:
                raise ValueError(f"kv_weight must be [{cache.kv_lora_rank}]")
            if kv_weight.data_ptr() % 16:
                kv_weight = kv_weight.clone()
        norm = head_norm(None, kv_weight, float(eps), float(weight_offset))
    result = None if q_pe is None else _result(q_pe, out, "q_pe")
    _no_gradients("mla_rotary_append", q_pe, kv_c, k_pe, kv_weight, out)
    with _on(dev):
        rc = _lib.load().wkv_mla_rotary_append(cache.descriptor(), kv_c.data_ptr(), kv_c.stride(0), k_pe.data_ptr(),
                                               k_pe.stride(0), slots.data_ptr(), *_rows(q_pe, result), norm, how, tokens,
                                               _stream(dev))
    if rc:
        _lib.check(rc, "mla_rotary_append")
    if out is not None:
        torch.autograd.graph.increment_version([out])
    return result
