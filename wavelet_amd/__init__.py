"""MI355X-native paged KV-cache decode path (gfx950 HIP kernels behind a C ABI).

Public surface (a drop-in for the KV path of the reference's inference engine):

* ``PagedKVCache`` / ``MLALatentCache`` -- per-layer caches with ``append``,
  ``gather`` and ``copy_blocks``;
* ``paged_decode_gqa`` / ``paged_decode_mla`` -- one decode step of attention;
  ``decode_order`` -- a step's longest-first dispatch order for the former,
  ``decode_plan`` -- its launch shape;
* ``paged_decode_gqa_grouped`` -- the same for GRPO groups, reading each
  group's shared prompt blocks through the caches and the members' own tokens
  streamed; ``grouped_decode_order`` -- its dispatch order;
* ``prefill_gqa`` -- varlen (chunked) prefill that appends the prompt's K/V
  and attends causally over the paged context;
* ``BlockManager`` -- host-side block allocation with ref-counted prefix
  sharing for GRPO groups;
* ``KVPool`` -- all layers' caches plus the block manager, with the engine's
  sleep / wake_up lifecycle and KV metrics;
* ``paged_tree_gqa`` -- attention of a tree of drafted tokens over the cache,
  and around it: ``extend_tables`` (a step's blocks, slots, positions and tree
  masks on the GPU), ``accept_tree`` (the path that the sampled tokens
  agree with) and ``PagedKVCache.compact`` (its keys and values moved together);
  ``KVPool.lend`` / ``settle`` / ``cancel`` -- the blocks and lengths of such steps,
  lent to the device and taken back (``StepState``);
* ``apply_rotary`` / ``rotary_frequencies`` -- rotary positions of queries and
  keys, with gradients;
* ``sample`` -- the token sampler after decode (temperature, min_p, top_k,
  top_p, repetition penalty; processed logprobs and the sampling mask).

Also, by module: ``wavelet_amd.plan`` -- a whole decode or prompt step over
every layer, built once and launched per step (``DecodeStep``,
``MLADecodeStep``, ``PrefillStep``, ``TreeStep``), and ``GraphDecodeStep``, the decode step
captured in one HIP graph; ``wavelet_amd.hf`` -- a transformers ``Cache`` over
a ``KVPool`` and the ``"wavelet_paged"`` attention implementation.
"""

from .attention import (decode_order, decode_plan, grouped_decode_order, paged_decode_gqa, paged_decode_gqa_grouped,
                        paged_decode_mla, paged_tree_gqa, prefill_gqa)
from .blocks import BlockManager
from .cache import MLALatentCache, PagedKVCache, validate_group_prefix, validate_tables
from .pool import KVPool
from .rotary import apply_rotary, rotary_frequencies
from .sampler import sample
from .step import Accepted, StepMaps, StepState, accept_tree, extend_tables

__all__ = [
    "Accepted",
    "BlockManager",
    "KVPool",
    "MLALatentCache",
    "PagedKVCache",
    "StepMaps",
    "StepState",
    "accept_tree",
    "apply_rotary",
    "decode_order",
    "grouped_decode_order",
    "decode_plan",
    "extend_tables",
    "paged_decode_gqa",
    "paged_decode_gqa_grouped",
    "paged_decode_mla",
    "paged_tree_gqa",
    "prefill_gqa",
    "rotary_frequencies",
    "sample",
    "validate_group_prefix",
    "validate_tables",
]
