"""A step's bookkeeping on the GPU: block tables, slots and positions from the request lengths, and the
accepted path of a verified tree.

The reference's engine makes its slot mapping and block tables on the host, between the steps of
``llm.generate`` (wavelet/inference/engine.py:887); ``BlockManager`` does so here. A step whose token
counts only the GPU knows -- drafted tokens of which some were accepted -- would have to wait for them
on the host. ``extend_tables`` and ``accept_tree`` keep lengths, tables and free blocks on the device
instead, in one launch (or two) per step for every layer.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import NamedTuple

import torch

from . import _lib
from .cache import _on, _require_cuda, _stream

MAX_BATCH = 2048  # WKV_STEP_MAX_BATCH
MAX_NODES = 256   # 64 * WKV_TREE_MAX_WORDS
MAX_DEPTH = 64    # WKV_TREE_MAX_DEPTH
NO_LIMIT = 2**31 - 1  # of a sequence's length


class StepMaps(NamedTuple):
    """What ``extend_tables`` makes of a step's lengths (all on the device)."""

    context_lens: torch.Tensor  # [B] int32: cached and new tokens (0: refused)
    cu_seqlens_q: torch.Tensor  # [B + 1] int32: the sequences' rows
    slot_mapping: torch.Tensor  # [max_tokens] int64
    positions: torch.Tensor     # [max_tokens] int64
    tree_mask: torch.Tensor | None  # [max_tokens, max_nodes / 64] int64
    refused: torch.Tensor       # [1] int32: sequences that got no slots
    held_blocks: torch.Tensor   # [B] int32 after the step
    taken: torch.Tensor         # [1] int32 after the step


class Accepted(NamedTuple):
    """A verified step's outcome (all on the device)."""

    accepted: torch.Tensor     # [B] int32
    path: torch.Tensor         # [B, max_depth] int32, -1 past the accepted nodes
    next_tokens: torch.Tensor  # [B] int64, -1 for a sequence that accepts nothing
    seq_lens: torch.Tensor     # [B] int32


@dataclass
class StepState:
    """The sequences of the next steps as the device carries them on (``KVPool.lend``): ``extend`` gives a
    step's tokens their blocks and slots, an accepted path's lengths go back into ``seq_lens`` and the token
    sampled after it into ``next_tokens`` (a sequence that accepts nothing keeps its own), and
    ``KVPool.settle`` hands tables and lengths to the block manager. No step takes a sequence past
    ``max_seq_len`` (the pool's ``max_model_len``; None: the tables' width alone is a limit)."""

    block_table: torch.Tensor  # [B, M] int32
    held_blocks: torch.Tensor  # [B] int32
    seq_lens: torch.Tensor     # [B] int32
    free_blocks: torch.Tensor  # [F] int32
    taken: torch.Tensor        # [1] int32
    block_size: int
    loan: object = None        # the block manager's
    max_seq_len: int | None = None
    next_tokens: torch.Tensor | None = None  # [B] int64: sampled, not cached yet: node 0 of the next step's trees

    def extend(self, new_lens: torch.Tensor, max_tokens: int, *, parents: torch.Tensor | None = None,
               max_nodes: int = 0, max_seq_len: int | None = None, out: StepMaps | None = None) -> StepMaps:
        """``extend_tables`` of this state, in place (``held_blocks`` and ``taken`` of the result are the state's), up
        to the state's ``max_seq_len`` or a lower one given here."""
        limits = [x for x in (self.max_seq_len, max_seq_len) if x is not None]
        if out is None:
            out = new_step_maps(self.block_table.shape[0], max_tokens, max_nodes, self.block_table.device)
        return extend_tables(self.block_table, self.held_blocks, self.seq_lens, new_lens, self.free_blocks, self.taken,
                             self.block_size, max_tokens, parents=parents, max_nodes=max_nodes,
                             max_seq_len=min(limits, default=None), out=out._replace(held_blocks=self.held_blocks, taken=self.taken))


def _vector(x: torch.Tensor, name: str, n: int | None, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    if isinstance(x, torch.Tensor) and x.device == device and x.dtype == dtype and x.dim() == 1 \
            and (n is None or x.shape[0] == n):
        return x.contiguous()
    _require_cuda(x, name, device)
    raise ValueError(f"{name} must be {dtype} [{'n' if n is None else n}] (got {x.dtype} {tuple(x.shape)})")


def _outputs(out, kinds, device: torch.device, what: str):
    """The caller's tensors, checked; kinds: (name, shape, dtype), a shape of None for none."""
    if len(out) != len(kinds):
        raise ValueError(f"out must be a {what}")
    for o, (name, shape, dtype) in zip(out, kinds):
        if (o is None) != (shape is None) or o is not None and (
                o.dtype != dtype or tuple(o.shape) != shape or not o.is_contiguous() or o.device != device):
            raise ValueError(f"out.{name} must be " +
                             ("None" if shape is None else f"a contiguous {dtype} {shape} tensor on {device}"))
    return out


def new_step_maps(batch: int, max_tokens: int, max_nodes: int, device: torch.device) -> StepMaps:
    """Tensors for ``extend_tables``'s ``out``, in one allocation (each alone costs the host 1.3 us)."""
    words, tail = max_nodes // 64, 3 * batch + 4 >> 1
    slots, positions, mask, ints = torch.empty((2 + words) * max_tokens + tail, dtype=torch.int64, device=device) \
        .split_with_sizes((max_tokens, max_tokens, words * max_tokens, tail))
    context, cu, held, refused, taken, _ = ints.view(torch.int32).split_with_sizes(
        (batch, batch + 1, batch, 1, 1, 2 * tail - 3 * batch - 3))
    return StepMaps(context, cu, slots, positions, mask.view(max_tokens, words) if words else None, refused, held, taken)


def _new_accepted(batch: int, max_depth: int, device: torch.device) -> Accepted:
    """The same for ``accept_tree``."""
    after, accepted, lens, path = torch.empty((4 + max_depth) * batch, dtype=torch.int32, device=device).split_with_sizes(
        (2 * batch, batch, batch, max_depth * batch))
    return Accepted(accepted, path.view(batch, max_depth), after.view(torch.int64), lens)


def extend_tables(block_table: torch.Tensor, held_blocks: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor,
                  free_blocks: torch.Tensor, taken: torch.Tensor, block_size: int, max_tokens: int, *,
                  parents: torch.Tensor | None = None, max_nodes: int = 0, max_seq_len: int | None = None,
                  out: StepMaps | None = None) -> StepMaps:
    """A step's blocks, slots and positions from its lengths, without the host.

    Sequence ``b`` (of at most 2,048) holds ``held_blocks[b]`` blocks, the leading entries of row ``b`` of
    ``block_table [B, M]`` (int32, written in place: its rows contiguous), and ``seq_lens[b]`` cached
    tokens, and brings ``new_lens[b]`` tokens (int32 ``[B]`` each). In batch order, each gets the blocks its
    tokens need beyond those it holds, the next of ``free_blocks`` (int32 ``[F]``) past the first
    ``taken`` (int32 ``[1]``). A sequence is refused, wholly, when it has too few table entries, rows
    (``max_tokens``) or nodes (``max_nodes``), would pass ``max_seq_len`` tokens (None: no limit), or needs
    blocks once those asked for are more than are free.

    The result's rows are the step's tokens, sequence by sequence (``cu_seqlens_q``), ``max_tokens`` of
    them: each token's slot and position, -1 for a refused sequence's and past the last. With ``max_nodes``
    (a multiple of 64 up to 256) the tokens are the nodes of one tree per sequence: ``parents [max_tokens]``
    int32 names each node's parent among its sequence's (an earlier node; -1: it follows the context
    directly), the position is the length plus the node's depth, and ``tree_mask`` holds the
    ancestors' bits for ``paged_tree_gqa``. ``context_lens`` counts cached and new tokens, the
    ``seq_lens`` of the step's attention (0 for a refused sequence: its rows give zeros); ``held_blocks``
    and ``taken`` are the state after the step. ``out``: preallocated results, whose ``held_blocks`` and
    ``taken`` may be the arguments themselves, so that a captured graph carries the state on.
    """
    _require_cuda(block_table, "block_table", block_table.device if isinstance(block_table, torch.Tensor) else None)
    dev = block_table.device
    if dev.type != "cuda":
        raise ValueError(f"block_table is on {dev}: extend_tables runs on the GPU")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1 or block_table.shape[1] < 1:
        raise ValueError("block_table must be int32 [B, max_blocks] with contiguous rows (it is written in place)")
    batch, width = block_table.shape
    if not 0 < batch <= MAX_BATCH:
        raise ValueError(f"a step takes 1 to {MAX_BATCH} sequences (got {batch})")
    if batch > 1 and block_table.stride(0) < width:
        raise ValueError("block_table rows must not overlap")
    held = _vector(held_blocks, "held_blocks", batch, torch.int32, dev)
    lens = _vector(seq_lens, "seq_lens", batch, torch.int32, dev)
    new = _vector(new_lens, "new_lens", batch, torch.int32, dev)
    free = _vector(free_blocks, "free_blocks", None, torch.int32, dev)
    taken = _vector(taken, "taken", 1, torch.int32, dev)
    max_tokens, max_nodes, block_size = int(max_tokens), int(max_nodes), int(block_size)
    if max_tokens < 0 or block_size <= 0:
        raise ValueError("max_tokens must be non-negative and block_size positive")
    max_seq_len = NO_LIMIT if max_seq_len is None else min(int(max_seq_len), NO_LIMIT)
    if max_seq_len < 0:
        raise ValueError(f"max_seq_len must be non-negative (got {max_seq_len})")
    if max_nodes % 64 or not 0 <= max_nodes <= MAX_NODES:
        raise ValueError(f"max_nodes must be a multiple of 64 up to {MAX_NODES} (got {max_nodes})")
    if (parents is None) != (max_nodes == 0):
        raise ValueError("a tree needs both parents and max_nodes")
    if parents is not None:
        parents = _vector(parents, "parents", max_tokens, torch.int32, dev)
    words = max_nodes // 64
    if out is None:
        m = new_step_maps(batch, max_tokens, max_nodes, dev)
    else:
        m = StepMaps(*_outputs(out, (("context_lens", (batch,), torch.int32), ("cu_seqlens_q", (batch + 1,), torch.int32),
                                     ("slot_mapping", (max_tokens,), torch.int64), ("positions", (max_tokens,), torch.int64),
                                     ("tree_mask", (max_tokens, words) if words else None, torch.int64),
                                     ("refused", (1,), torch.int32), ("held_blocks", (batch,), torch.int32),
                                     ("taken", (1,), torch.int32)), dev, "StepMaps"))
    with _on(dev):
        rc = _lib.load().wkv_extend_tables_limited(
            block_table.data_ptr(), max(block_table.stride(0), width), width, held.data_ptr(), lens.data_ptr(),
            new.data_ptr(), batch, block_size, free.data_ptr() or None, free.shape[0], taken.data_ptr(), max_tokens,
            max_seq_len, parents.data_ptr() if words else None, words, m.held_blocks.data_ptr(), m.taken.data_ptr(),
            m.context_lens.data_ptr(), m.cu_seqlens_q.data_ptr(), m.slot_mapping.data_ptr(), m.positions.data_ptr(),
            m.tree_mask.data_ptr() if words else None, m.refused.data_ptr(), _stream(dev))
    _lib.check(rc, "extend_tables")
    return m


def accept_tree(draft_tokens: torch.Tensor, parents: torch.Tensor, target_tokens: torch.Tensor,
                cu_seqlens_q: torch.Tensor, seq_lens: torch.Tensor, context_lens: torch.Tensor, max_depth: int, *,
                pending: torch.Tensor | None = None, out: Accepted | None = None) -> Accepted:
    """The drafted tokens of a verified tree that agree with the sampled ones.

    ``draft_tokens [T]`` int64 and ``parents [T]`` int32 are the trees' nodes, sequence by sequence
    (``cu_seqlens_q``), as for ``extend_tables``; ``target_tokens [T]`` int64 is the token sampled after each
    node (``sample`` over the nodes' logits). Node 0 of a sequence -- the token of the step before -- is
    accepted; an accepted node's path goes on to its first child whose token is the one sampled after
    it, up to ``max_depth`` (at most 64) nodes. ``next_tokens`` is what was sampled after the last.
    ``seq_lens`` are the lengths before the step, and the result's those with the accepted tokens
    (``out.seq_lens`` may be the argument); ``PagedKVCache.compact`` moves their keys and values there. A
    sequence without nodes or with ``context_lens`` 0 (refused by ``extend_tables``) accepts nothing
    (``next_tokens`` -1). ``pending [B]`` int64, written in place: the token that each sequence goes on with,
    ``next_tokens`` where anything was accepted, else what it was.
    """
    _require_cuda(cu_seqlens_q, "cu_seqlens_q", cu_seqlens_q.device if isinstance(cu_seqlens_q, torch.Tensor) else None)
    dev = cu_seqlens_q.device
    if dev.type != "cuda":
        raise ValueError(f"cu_seqlens_q is on {dev}: accept_tree runs on the GPU")
    if cu_seqlens_q.dtype != torch.int32 or cu_seqlens_q.dim() != 1 or cu_seqlens_q.shape[0] < 1:
        raise ValueError("cu_seqlens_q must be int32 [B + 1]")
    batch = cu_seqlens_q.shape[0] - 1
    cu = cu_seqlens_q.contiguous()
    draft = _vector(draft_tokens, "draft_tokens", None, torch.int64, dev)
    rows = draft.shape[0]
    parents = _vector(parents, "parents", rows, torch.int32, dev)
    target = _vector(target_tokens, "target_tokens", rows, torch.int64, dev)
    lens = _vector(seq_lens, "seq_lens", batch, torch.int32, dev)
    context = _vector(context_lens, "context_lens", batch, torch.int32, dev)
    max_depth = int(max_depth)
    if not 1 <= max_depth <= MAX_DEPTH:
        raise ValueError(f"max_depth must be in [1, {MAX_DEPTH}] (got {max_depth})")
    if pending is not None and (_vector(pending, "pending", batch, torch.int64, dev) is not pending):
        raise ValueError("pending must be contiguous (it is written in place)")
    if out is None:
        a = _new_accepted(batch, max_depth, dev)
    else:
        a = Accepted(*_outputs(out, (("accepted", (batch,), torch.int32), ("path", (batch, max_depth), torch.int32),
                                     ("next_tokens", (batch,), torch.int64), ("seq_lens", (batch,), torch.int32)), dev,
                               "Accepted"))
    if batch == 0:
        return a
    with _on(dev):
        rc = _lib.load().wkv_accept_tree_pending(
            draft.data_ptr(), parents.data_ptr(), target.data_ptr(), rows, cu.data_ptr(), lens.data_ptr(),
            context.data_ptr(), batch, max_depth, a.accepted.data_ptr(), a.path.data_ptr(), a.next_tokens.data_ptr(),
            a.seq_lens.data_ptr(), pending.data_ptr() if pending is not None else None, _stream(dev))
    _lib.check(rc, "accept_tree")
    return a
