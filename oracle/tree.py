"""A step of drafted tokens restated in numpy (oracle; tests only): the rotation of queries and keys,
the step's block tables and slots, attention of a tree over the paged cache, the accepted path, and
the move of its keys and values. Plain loops over sequences and nodes, float64 where values are computed.

Pinned in tests/test_tree_oracle.py: a chain's attention is ``paged.prefill_gqa``'s, a chain's slots are
``BlockManager.append_slots``'s, the rotation keeps norms and its inverse undoes it, and the move is
``paged.gather`` followed by ``paged.append_bf16`` / ``append_fp8``.
"""

from __future__ import annotations

import numpy as np

from . import fp8, paged


def rotary(x, positions, inv_freq, *, interleaved=False, scale=1.0, inverse=False):
    """Rows ``x [T, H, D]`` with pair ``i`` of every head turned by ``positions[t] * inv_freq[i]`` and
    multiplied by ``scale`` (float64). Pair ``i`` is dims ``(2i, 2i + 1)`` if interleaved, else
    ``(i, i + R / 2)``, ``R = 2 len(inv_freq)``; dims from ``R`` on stay as they are."""
    x = np.asarray(x, np.float64)
    half = len(inv_freq)
    angle = np.asarray(positions, np.float64)[:, None] * np.asarray(inv_freq, np.float64)
    c, s = np.cos(angle)[:, None] * scale, np.sin(angle)[:, None] * scale
    s = -s if inverse else s
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y = x.copy()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def parent_of(parents, i: int) -> int:
    """Node ``i``'s parent among its sequence's nodes, or -1 (an entry that is no earlier node counts as none)."""
    p = int(parents[i])
    return p if 0 <= p < i else -1


def ancestors(parents, i: int) -> list[int]:
    """Node ``i`` and the nodes above it, rising."""
    out = [i]
    while parent_of(parents, out[-1]) >= 0:
        out.append(parent_of(parents, out[-1]))
    return out[::-1]


def masks(parents, words: int) -> np.ndarray:
    """``[n, words]`` int64: the bits of every node's ancestors, itself among them."""
    out = np.zeros((len(parents), words), np.uint64)
    for i in range(len(parents)):
        for j in ancestors(parents, i):
            out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out.view(np.int64)


def extend_tables(block_table, held_blocks, seq_lens, new_lens, free_blocks, taken, block_size, max_tokens, *,
                  parents=None, max_nodes=0, max_seq_len=2**31 - 1):
    """The step's tables (see ``wavelet_amd.extend_tables``): a dict of its outputs, ``block_table`` a copy."""
    table = np.array(block_table, np.int32)
    b, width = table.shape
    length = np.maximum(np.asarray(seq_lens, np.int64), 0)
    new = np.maximum(np.asarray(new_lens, np.int64), 0)
    held = np.maximum(np.asarray(held_blocks, np.int64), 0)
    words = max_nodes // 64
    cu = np.minimum(np.concatenate([[0], np.cumsum(new)]), max_tokens).astype(np.int32)
    context = length.copy()
    slots = np.full(max_tokens, -1, np.int64)
    positions = np.full(max_tokens, -1, np.int64)
    mask = np.zeros((max_tokens, words), np.int64)
    at, asked, given, refused, row = int(taken), int(taken), 0, 0, 0
    held_out = held.copy()
    for i in range(b):
        n = int(new[i])
        start, row = row, row + n
        if n == 0:
            continue
        total = -(-int(length[i] + n) // block_size)
        fits = total <= width and length[i] + n <= max_seq_len and row <= max_tokens and (words == 0 or n <= max_nodes)
        need = max(total - int(held[i]), 0) if fits else 0
        asked += need  # a sequence that is refused its blocks still stands in the queue
        if not fits or (need > 0 and asked > len(free_blocks)):
            context[i] = 0
            refused += 1
            continue
        for k in range(need):
            table[i, held[i] + k] = free_blocks[asked - need + k]
        held_out[i] += need
        given += need
        context[i] = length[i] + n
        for j in range(n):
            pos = int(length[i]) + j
            if table[i, pos // block_size] >= 0:  # else the table holds no block there
                slots[start + j] = int(table[i, pos // block_size]) * block_size + pos % block_size
            if words:
                up = ancestors(parents[start:start + n], j)
                positions[start + j] = int(length[i]) + len(up) - 1
                mask[start + j] = masks(parents[start:start + n][:j + 1], words)[j]
            else:
                positions[start + j] = pos
    return dict(block_table=table, held_blocks=held_out.astype(np.int32), taken=at + given,
                context_lens=context.astype(np.int32), cu_seqlens_q=cu, slot_mapping=slots, positions=positions,
                tree_mask=mask, refused=refused)


def accept_tree(draft_tokens, parents, target_tokens, cu_seqlens_q, seq_lens, context_lens, max_depth):
    """``(accepted, path, next_tokens, seq_lens)`` as ``wavelet_amd.accept_tree`` documents them."""
    b = len(cu_seqlens_q) - 1
    accepted, nxt = np.zeros(b, np.int32), np.full(b, -1, np.int64)
    path = np.full((b, max_depth), -1, np.int32)
    for i in range(b):
        q0, n = int(cu_seqlens_q[i]), int(cu_seqlens_q[i + 1] - cu_seqlens_q[i])
        if n == 0 or context_lens[i] <= 0:
            continue
        par = parents[q0:q0 + n]
        way = [0]
        while len(way) < max_depth:
            want = target_tokens[q0 + way[-1]]
            on = [j for j in range(way[-1] + 1, n) if parent_of(par, j) == way[-1] and draft_tokens[q0 + j] == want]
            if not on:
                break
            way.append(on[0])
        accepted[i], nxt[i] = len(way), target_tokens[q0 + way[-1]]
        path[i, :len(way)] = way
    return accepted, path, nxt, (np.maximum(np.asarray(seq_lens), 0) + accepted).astype(np.int32)


def compact(k, v, k_scale, v_scale, block_table, seq_lens, path, accepted) -> None:
    """The tokens at positions ``seq_lens[i] + path[i, j]`` to ``seq_lens[i] + j``, in place: those that change
    their place are read together, then appended (fp8: their exact values, as ``append_fp8`` codes them). One
    whose old or new position has no block is left out."""
    bs = v.shape[-1]
    nb, h, d = v.shape[:3]
    for i in range(len(seq_lens)):
        row = np.asarray(block_table[i])

        def slot(p):
            blk = int(row[p // bs]) if 0 <= p < len(row) * bs else -1
            return blk * bs + p % bs if 0 <= blk < nb else -1

        at = max(int(seq_lens[i]), 0)
        places = [(slot(at + int(path[i, j])), slot(at + j)) for j in range(int(accepted[i]))
                  if path[i, j] != j and path[i, j] >= 0]
        places = np.array([p for p in places if min(p) >= 0]).reshape(-1, 2)
        if not len(places):
            continue
        src, dst = places.T
        kl = np.ascontiguousarray(paged.k_logical(k)[src // bs, src % bs]).reshape(len(src), h, d)
        vl = np.ascontiguousarray(paged.v_logical(v)[src // bs, src % bs])
        if k_scale is None:
            paged.append_bf16(k, v, kl, vl, dst)
        else:
            kf = fp8.dequantize(kl, k_scale[src // bs][:, :, None])
            vf = fp8.dequantize(vl, v_scale[src // bs][:, :, None])
            paged.append_fp8(k, v, k_scale, v_scale, paged.f32_to_bf16(kf), paged.f32_to_bf16(vf), dst)


def tree_gqa(q, k_vals, v_vals, block_table, seq_lens, cu_seqlens_q, tree_mask, scale, *, sinks=None, num_blocks=None):
    """Attention of every sequence's last ``n_i = cu[i + 1] - cu[i]`` tokens (float64): row ``j`` sees the
    ``seq_lens[i] - n_i`` tokens before them and those of the ``n_i`` whose bit its mask sets. ``k_vals`` /
    ``v_vals`` are logical ``[NB, BS, Hkv, D]`` values; keys of a block outside the cache are seen by no row,
    and a row that sees none gives zeros."""
    t, hq, d = q.shape
    nb, bs, hkv, _ = k_vals.shape
    g = hq // hkv
    out = np.zeros((t, hq, d))
    for i in range(len(seq_lens)):
        q0, n, length = int(cu_seqlens_q[i]), int(cu_seqlens_q[i + 1] - cu_seqlens_q[i]), int(seq_lens[i])
        if n == 0 or length <= 0:
            continue
        pos = np.arange(length)
        blk = np.asarray(block_table[i], np.int64)[pos // bs]
        real = (blk >= 0) & (blk < nb)
        kk = k_vals[np.where(real, blk, 0), pos % bs].astype(np.float64)
        vv = v_vals[np.where(real, blk, 0), pos % bs].astype(np.float64)
        for j in range(n):
            bits = np.asarray(tree_mask[q0 + j]).view(np.uint64)
            node = pos - (length - n)
            seen = real & ((node < 0) | [x >= 0 and bool(bits[x // 64] >> np.uint64(x % 64) & np.uint64(1)) for x in node])
            if not seen.any():
                continue
            for h in range(hq):
                s = kk[seen, h // g] @ q[q0 + j, h].astype(np.float64) * scale
                m = s.max() if sinks is None else max(s.max(), float(sinks[h]))
                e = np.exp(s - m)
                den = e.sum() + (0.0 if sinks is None else np.exp(float(sinks[h]) - m))
                out[q0 + j, h] = (e / den) @ vv[seen, h // g]
    return out
