"""The measured calls of a step of drafted tokens: what it needs on the GPU, operator by operator.

A serving loop that drafts several tokens per sequence (a tree of continuations, or one chain)
runs, per step: ``extend_tables`` (blocks, slots, positions and the tree's masks from the request
lengths), per layer ``apply_rotary`` and ``paged_tree_gqa`` (the drafted tokens over the cache),
``accept_tree`` on the sampled tokens, and per layer ``PagedKVCache.compact`` (the accepted path's
keys and values moved together). ``apply_rotary`` also serves prompts, single tokens and training.

With ``own`` false the same results come from elementary torch operations in 32 bits (64 where an
angle needs them). Sizes are the model layouts, batches and context ranges of this repository's
benchmark and tests; block tables are dealt from a shuffled pool, as a running engine's are.
"""

from __future__ import annotations

import math

import torch

own = False

# layout: query heads, KV heads, head dim
MODELS = {
    "qwen2.5-0.5b": (14, 2, 64),
    "qwen3-0.6b": (16, 8, 128),
    "qwen3-4b": (32, 8, 128),
    "qwen2.5-7b": (28, 4, 128),
    "qwen3-30b-a3b": (32, 4, 128),
}


def listed() -> list[dict]:
    return [
        # The step of a rollout batch: 64 sequences, each with a tree of 16 drafted tokens.
        dict(name="tables_step", kind="tables", batch=64, ctx_lo=500, ctx_hi=4096, new_lo=16, new_hi=16, block=16,
             tree=True, short=False),
        # A batch of prompts admitted at once: every block of every prompt comes from the free list.
        dict(name="tables_prompts", kind="tables", batch=64, ctx_lo=0, ctx_hi=0, new_lo=301, new_hi=2048, block=16,
             tree=False, short=False),
        # One token of one sequence at a far position: a decode step's latency.
        dict(name="rotary_token", kind="rotary", model="qwen3-4b", tokens=1, rotary=128, inter=False, dtype="bf16",
             top=131072, base=1e6, factor=1.0, grad=False),
        # The prompts of a step: 16,384 tokens of whole rotated heads.
        dict(name="rotary_prompts", kind="rotary", model="qwen3-4b", tokens=16384, rotary=128, inter=False,
             dtype="bf16", top=32768, base=1e6, factor=1.0, grad=False),
        # A training batch of odd size: forward and backward, adjacent pairs, half of each head
        # rotated, positions divided for a long context.
        dict(name="rotary_train", kind="rotary", model="qwen2.5-7b", tokens=4097, rotary=64, inter=True, dtype="bf16",
             top=32768, base=1e4, factor=4.0, grad=True),
        # One sequence of a small model with eight drafted tokens: an interactive request.
        dict(name="tree_one", kind="tree", model="qwen2.5-0.5b", kv="bf16", batch=1, ctx_lo=700, ctx_hi=700,
             new_lo=8, new_hi=8, block=16),
        # The rollout batch's trees over 4,096 tokens each.
        dict(name="tree_batch", kind="tree", model="qwen3-4b", kv="bf16", batch=64, ctx_lo=4096, ctx_hi=4096,
             new_lo=16, new_hi=16, block=16),
        # Few long ragged contexts with wide ragged trees, fp8 KV, seven query heads per KV head.
        dict(name="tree_long_fp8", kind="tree", model="qwen2.5-7b", kv="fp8_e4m3", batch=6, ctx_lo=3001,
             ctx_hi=24001, new_lo=5, new_hi=63, block=32),
        # The verified tokens of a large batch with wide trees.
        dict(name="accept_batch", kind="accept", batch=256, new_lo=64, new_hi=64, depth=16),
        # A few requests' trees of odd sizes.
        dict(name="accept_few", kind="accept", batch=4, new_lo=3, new_hi=31, depth=8),
        # The accepted paths of a rollout batch moved together, one layer, bf16.
        dict(name="compact_batch", kind="compact", model="qwen3-4b", kv="bf16", batch=64, ctx_lo=65, ctx_hi=500,
             new_lo=16, new_hi=16, depth=8, block=16),
        # The same with fp8 KV: moved tokens are encoded again at their new blocks' scales.
        dict(name="compact_fp8", kind="compact", model="qwen2.5-7b", kv="fp8_e4m3", batch=33, ctx_lo=65, ctx_hi=500,
             new_lo=9, new_hi=63, depth=12, block=16),
    ]


_MAX_TREE_BYTES = 1.1e9   # cached bytes of the largest drawn tree step (the listed batch's)
_MAX_TREE_PAIRS = 1.4e8   # its scored pairs of a query head's row and a key
_MAX_ROTARY = 16384 * 40 * 128  # values of the largest drawn rotation


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _range(rng, lo: int, hi: int) -> tuple[int, int]:
    top = _log_int(rng, lo, hi)
    return rng.choice([top, max(lo, top // 3), lo]), top


def draw(rng) -> dict:
    kind = rng.choice(["tables", "rotary", "rotary", "tree", "tree", "tree", "accept", "compact", "compact"])
    if kind == "tables":
        tree = bool(rng.random() < 0.6)
        batch = _log_int(rng, 1, 512)
        n_lo, n_hi = _range(rng, 1, 128) if tree else _range(rng, 1, max(1, min(4096, 131072 // batch)))
        c_lo, c_hi = rng.choice([(0, 0), _range(rng, 1, 16384)])
        return dict(kind=kind, batch=batch, ctx_lo=c_lo, ctx_hi=c_hi, new_lo=n_lo, new_hi=n_hi,
                    block=rng.choice([16, 16, 32, 64]), tree=tree, short=bool(rng.random() < 0.3))
    if kind == "rotary":
        model = rng.choice(sorted(MODELS))
        hq, hkv, d = MODELS[model]
        grad = bool(rng.random() < 0.4)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        cost = (hq + hkv) * d / 128 * (2 if grad else 1) * (2 if dtype == "fp32" else 1)
        tokens = _log_int(rng, 1, max(1, int(_MAX_ROTARY / 128 / cost)))
        return dict(kind=kind, model=model, tokens=tokens, rotary=rng.choice([d, d, d // 2, d // 4, 2 * rng.randint(1, d // 2)]),
                    inter=bool(rng.random() < 0.4), dtype=dtype, top=_log_int(rng, 64, 1 << 20),
                    base=rng.choice([1e4, 1e6]), factor=rng.choice([1.0, 4.0]), grad=grad)
    if kind == "tree":
        model = rng.choice(sorted(MODELS))
        hq, hkv, d = MODELS[model]
        c_lo, c_hi = _range(rng, 1, 32768)
        n_lo, n_hi = _range(rng, 1, 128)
        case = dict(kind=kind, model=model, kv=rng.choice(["bf16", "bf16", "fp8_e4m3"]), batch=_log_int(rng, 1, 64),
                    ctx_lo=c_lo, ctx_hi=c_hi, new_lo=n_lo, new_hi=n_hi, block=rng.choice([16, 16, 32, 64]))
        while (case["batch"] * (c_hi + n_hi) * hkv * d * 4 > _MAX_TREE_BYTES
               or case["batch"] * (c_hi + n_hi) * n_hi * hq > _MAX_TREE_PAIRS):
            if case["batch"] > 1:
                case["batch"] //= 2
            else:
                n_hi = case["new_hi"] = max(1, n_hi // 2)
                case["new_lo"] = min(case["new_lo"], n_hi)
        return case
    n_lo, n_hi = _range(rng, 1, 128)
    if kind == "accept":
        return dict(kind=kind, batch=_log_int(rng, 1, 256), new_lo=n_lo, new_hi=n_hi, depth=rng.randint(1, 64))
    c_lo, c_hi = _range(rng, 1, 600)
    return dict(kind=kind, model=rng.choice(sorted(MODELS)), kv=rng.choice(["bf16", "fp8_e4m3"]),
                batch=_log_int(rng, 1, 64), ctx_lo=c_lo, ctx_hi=c_hi, new_lo=n_lo, new_hi=n_hi,
                depth=rng.randint(1, 24), block=rng.choice([16, 16, 32, 64]))


# --------------------------------------------------------------------------- sizes

def _spread(lo: int, hi: int, n: int) -> list[int]:
    """n lengths spread evenly over [lo, hi]: the same for every seed (which sequence has which is not)."""
    return [lo + (hi - lo) * i // (n - 1) if n > 1 else hi for i in range(n)]


def _lens(case: dict) -> tuple[list[int], list[int]]:
    """Context and new lengths; the new ones run the other way, so that short contexts have wide trees too."""
    return _spread(case["ctx_lo"], case["ctx_hi"], case["batch"]), _spread(case["new_lo"], case["new_hi"], case["batch"])[::-1]


def _words(case: dict) -> int:
    return -(-case["new_hi"] // 64)


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "rotary":
        hq, hkv, d = MODELS[case["model"]]
        esz = 4 if case["dtype"] == "fp32" else 2
        values = case["tokens"] * (hq + hkv) * d * (2 if case["grad"] else 1)
        turned = case["tokens"] * (hq + hkv) * case["rotary"] * (2 if case["grad"] else 1)
        return {"bytes": 2 * values * esz + case["tokens"] * 8, "flops": 3 * turned}
    if kind == "accept":
        t = sum(_spread(case["new_lo"], case["new_hi"], case["batch"]))
        return {"bytes": t * (8 + 8 + 4) + case["batch"] * (4 * 5 + 8 + 4 * case["depth"]), "flops": 0}
    ctx, new = _lens(case)
    t, b, block = sum(new), case["batch"], case["block"]
    if kind == "tables":
        taken = sum(-(-(c + n) // block) - -(-c // block) for c, n in zip(ctx, new))
        touched = sum((c + n - 1) // block - c // block + 1 for c, n in zip(ctx, new) if n)
        return {"bytes": t * (8 + 8 + ((4 + 8 * _words(case)) if case["tree"] else 0)) + 4 * (touched + taken) + 24 * b,
                "flops": 0}
    hq, hkv, d = MODELS[case["model"]]
    esz = 2 if case["kv"] == "bf16" else 1
    if kind == "tree":
        pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))  # at most this many of a chain; a tree has fewer
        kv = (sum(ctx) + t) * 2 * hkv * d * esz
        append = t * 2 * hkv * d * 2 * 2 if case["kv"] == "bf16" else 0
        return {"bytes": kv + append + t * (2 * hq * d * 2 + 8 * _words(case)), "flops": 4 * pairs * hq * d}
    moved = sum(min(case["depth"], n) for n in new)  # at most: a path that keeps its place moves nothing
    return {"bytes": 2 * moved * 2 * hkv * d * esz + 4 * b * (2 + case["depth"]), "flops": 0}


# --------------------------------------------------------------------------- inputs

def _device() -> torch.device:
    return torch.device("cuda", torch.cuda.current_device())


def _gens(seed: int):
    g = torch.Generator(device=_device())
    g.manual_seed(seed)
    h = torch.Generator()
    h.manual_seed(seed)
    return g, h


def _i32(x) -> torch.Tensor:
    return torch.as_tensor(x, dtype=torch.int32).to(_device())


def _normal(gen, shape, dtype=torch.bfloat16) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype, device=_device()).normal_(generator=gen)


def _cumulative(new: list[int]) -> torch.Tensor:
    cu = torch.zeros(len(new) + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(torch.tensor(new), 0)
    return cu


def _trees(h, new: list[int]) -> torch.Tensor:
    """Parents within each sequence: node 0 the root, each other node under one of the eight before it."""
    out = []
    for n in new:
        i = torch.arange(n)
        lo = (i - 8).clamp_min(0)
        p = lo + (torch.rand(n, generator=h) * (i - lo)).floor().to(torch.int64)
        p[0] = -1
        out.append(p)
    return torch.cat(out).to(torch.int32)


def _masks(parents: torch.Tensor, new: list[int], words: int) -> torch.Tensor:
    """The ancestors of every node, itself among them, as bits of `words` 64-bit words."""
    out = torch.zeros((len(parents), words), dtype=torch.int64)
    at = 0
    for n in new:
        p = parents[at:at + n].tolist()
        rows = []
        for i in range(n):
            rows.append((rows[p[i]] if p[i] >= 0 else 0) | 1 << i)
        for w in range(words):
            part = [r >> 64 * w & (1 << 64) - 1 for r in rows]
            out[at:at + n, w] = torch.tensor([x - (1 << 64) if x >> 63 else x for x in part], dtype=torch.int64)
        at += n
    return out


def _shuffled(case: dict, h) -> tuple[list[int], list[int]]:
    ctx, new = _lens(case)
    order = torch.randperm(len(ctx), generator=h).tolist()
    return [ctx[i] for i in order], [new[i] for i in order]


def _dealt(h, need: list[int]) -> torch.Tensor:
    """A block table dealt from a shuffled pool of just as many blocks."""
    perm = torch.randperm(sum(need), generator=h).to(torch.int32)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    return table


def _fill_kv(gen, blocks: int, hkv: int, d: int, block: int, kv: str) -> list:
    """One layer's cache in the library's documented layout: K [N, H, D/x, B, x], V [N, H, D, B], scales."""
    if kv == "bf16":
        return [_normal(gen, (blocks, hkv, d // 8, block, 8)), _normal(gen, (blocks, hkv, d, block)), None, None]
    out = []
    for shape in ((blocks, hkv, d // 16, block, 16), (blocks, hkv, d, block)):
        x = _normal(gen, shape, torch.float32)
        e = torch.randint(-7, -3, (blocks, hkv), generator=gen, device=_device())
        s = torch.ldexp(torch.ones((blocks, hkv), device=_device()), e)
        x = x / s.view(blocks, hkv, *([1] * (len(shape) - 2)))
        out.append((x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), s))
    return [out[0][0], out[1][0], out[0][1], out[1][1]]


def _tables_inputs(case: dict, seed: int) -> dict:
    _, h = _gens(seed)
    b, block = case["batch"], case["block"]
    ctx, new = _shuffled(case, h)
    # a step's tree may have left a sequence a block more than its tokens fill
    held = [-(-c // block) + int(torch.randint(0, 2, (1,), generator=h)) for c in ctx]
    grown = [max(x, -(-(c + n) // block)) for x, c, n in zip(held, ctx, new)]
    table = torch.full((b, max(grown) + 2), -1, dtype=torch.int32)
    fresh = sum(grown) - sum(held)
    spare = fresh // 2 if case["short"] else fresh + 7
    perm = torch.randperm(sum(held) + spare + 5, generator=h).to(torch.int32)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = perm[at:at + n]
        at += n
    parents = _trees(h, new).to(_device()) if case["tree"] else None
    rows = -(-sum(new) // 64) * 64  # the step's row buffers, a little longer than its tokens
    if parents is not None:
        parents = torch.cat([parents, torch.full((rows - len(parents),), -1, dtype=torch.int32, device=_device())])
    return dict(table=table.to(_device()), held=_i32(held), seq_lens=_i32(ctx), new_lens=_i32(new),
                free=perm[at:].to(_device()), taken=_i32([5]), rows=rows, parents=parents, block=block,
                nodes=64 * _words(case) if case["tree"] else 0)


def _frequencies(case: dict, dtype=torch.float64) -> torch.Tensor:
    r = case["rotary"]
    i = torch.arange(0, r, 2, dtype=dtype, device=_device())
    return 1.0 / (case["base"] ** (i / r) * case["factor"])


def _rotary_inputs(case: dict, seed: int) -> dict:
    gen, h = _gens(seed)
    hq, hkv, d = MODELS[case["model"]]
    t = case["tokens"]
    dt = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[case["dtype"]]
    start = int(torch.randint(0, case["top"], (1,), generator=h))
    pos = (start + torch.arange(t, device=_device())) % case["top"]
    # q, k and v lie side by side, as a fused projection leaves them
    x = _normal(gen, (t, (hq + 2 * hkv) * d), dt)
    q, k, _ = x.split([hq * d, hkv * d, hkv * d], 1)
    out = dict(q=q.view(t, hq, d), k=k.view(t, hkv, d), pos=pos, freq=_frequencies(case),
               scale=1.0 if case["factor"] == 1.0 else 0.1 * math.log(case["factor"]) + 1.0)
    if case["grad"]:
        out.update(gq=_normal(gen, (t, hq, d), dt), gk=_normal(gen, (t, hkv, d), dt))
    return out


def _tree_inputs(case: dict, seed: int) -> dict:
    gen, h = _gens(seed)
    hq, hkv, d = MODELS[case["model"]]
    block = case["block"]
    ctx, new = _shuffled(case, h)
    lens = [c + n for c, n in zip(ctx, new)]
    table = _dealt(h, [-(-n // block) for n in lens])
    t = sum(new)
    mask = _masks(_trees(h, new), new, _words(case))
    slots = [table[i, (p := torch.arange(c, c + n)) // block].to(torch.int64) * block + p % block
             for i, (c, n) in enumerate(zip(ctx, new))]
    blocks = sum(-(-n // block) for n in lens)
    out = dict(table=table.to(_device()), seq_lens=_i32(lens), cu=_cumulative(new).to(_device()),
               mask=mask.to(_device()), kv=_fill_kv(gen, blocks, hkv, d, block, case["kv"]), blocks=blocks,
               q=_normal(gen, (t, hq, d)), scale=d ** -0.5, longest=max(new), context=max(lens), block=block)
    if case["kv"] == "bf16":  # fp8: the drafted tokens are in the cache already
        out.update(key=_normal(gen, (t, hkv, d)), value=_normal(gen, (t, hkv, d)), slots=torch.cat(slots).to(_device()))
    return out


def _accept_inputs(case: dict, seed: int) -> dict:
    _, h = _gens(seed)
    new = _spread(case["new_lo"], case["new_hi"], case["batch"])
    new = [new[i] for i in torch.randperm(len(new), generator=h).tolist()]
    t = sum(new)
    # few different tokens, so that paths of several nodes are accepted
    draft = torch.randint(0, 3, (t,), generator=h) * 50021 + 17
    target = torch.randint(0, 3, (t,), generator=h) * 50021 + 17
    lens = torch.randint(0, 4096, (len(new),), generator=h)
    return dict(draft=draft.to(_device()), target=target.to(_device()), parents=_trees(h, new).to(_device()),
                cu=_cumulative(new).to(_device()), seq_lens=_i32(lens), context_lens=_i32(lens + torch.tensor(new)),
                depth=case["depth"], longest=max(new))


def _compact_inputs(case: dict, seed: int) -> dict:
    gen, h = _gens(seed)
    _, hkv, d = MODELS[case["model"]]
    block, depth = case["block"], case["depth"]
    ctx, new = _shuffled(case, h)
    table = _dealt(h, [-(-(c + n) // block) for c, n in zip(ctx, new)])
    path = torch.full((len(new), depth), -1, dtype=torch.int32)
    count = []
    for i, n in enumerate(new):
        # node 0, then nodes in rising order, as a path down a tree has them
        a = 1 + int(torch.randint(0, min(depth, n), (1,), generator=h))
        rest = torch.randperm(n - 1, generator=h)[:a - 1].sort().values + 1
        path[i, :a] = torch.cat([torch.zeros(1, dtype=torch.int64), rest]).to(torch.int32)
        count.append(a)
    blocks = sum(-(-(c + n) // block) for c, n in zip(ctx, new))
    return dict(table=table.to(_device()), seq_lens=_i32(ctx), path=path.to(_device()), accepted=_i32(count),
                kv=_fill_kv(gen, blocks, hkv, d, block, case["kv"]), blocks=blocks, block=block)


_INPUTS = {"tables": _tables_inputs, "rotary": _rotary_inputs, "tree": _tree_inputs, "accept": _accept_inputs,
           "compact": _compact_inputs}


def prepare(case: dict, seed: int) -> dict:
    s = _INPUTS[case["kind"]](case, seed)
    s.update(kind=case["kind"], fp8=case.get("kv") == "fp8_e4m3", inter=case.get("inter", False))
    if s["kind"] == "rotary" and case["grad"]:
        s["q"].requires_grad_(True)
        s["k"].requires_grad_(True)
    if own and "kv" in s:  # the layer's cache, which a serving program keeps
        from wavelet_amd import PagedKVCache

        _, hkv, d = MODELS[case["model"]]
        c = s["cache"] = PagedKVCache(s["blocks"], s["block"], hkv, d, kv_dtype=case["kv"], device=_device())
        for name, x in zip(("k", "v", "k_scale", "v_scale"), s.pop("kv")):
            if x is not None:
                getattr(c, name).copy_(x)
    return s


# --------------------------------------------------------------------------- the framework's calls

def _contents(k, v, ks, vs) -> list:
    """A cache as the values that it holds: bf16 tensors, or fp8 values with their blocks' scales."""
    return [k, v] if ks is None else [k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), ks, vs]


def _run_own(s: dict) -> list:
    import wavelet_amd as w

    if s["kind"] == "tables":
        m = w.extend_tables(s["table"], s["held"], s["seq_lens"], s["new_lens"], s["free"], s["taken"], s["block"],
                            s["rows"], parents=s["parents"], max_nodes=s["nodes"])
        return [s["table"], m.held_blocks, m.taken, m.context_lens, m.cu_seqlens_q, m.slot_mapping, m.positions,
                m.refused] + ([m.tree_mask] if s["nodes"] else [])
    if s["kind"] == "rotary":
        q, k = w.apply_rotary(s["q"], s["k"], s["pos"], s["freq"], interleaved=s["inter"], scale=s["scale"])
        if "gq" not in s:
            return [q, k]
        gq, gk = torch.autograd.grad([q, k], [s["q"], s["k"]], [s["gq"], s["gk"]])
        return [q.detach(), k.detach(), gq, gk]
    if s["kind"] == "tree":
        new = dict(key=s["key"], value=s["value"], slot_mapping=s["slots"]) if "key" in s else {}
        out = w.paged_tree_gqa(s["q"], s["cache"], s["table"], s["seq_lens"], s["cu"], s["mask"], s["scale"],
                               max_query_len=s["longest"], max_seq_len=s["context"], **new)
        return [out] + ([s["cache"].k, s["cache"].v] if new else [])
    if s["kind"] == "accept":
        return list(w.accept_tree(s["draft"], s["parents"], s["target"], s["cu"], s["seq_lens"], s["context_lens"],
                                  s["depth"]))
    c = s["cache"]
    c.compact(s["table"], s["seq_lens"], s["path"], s["accepted"])
    return _contents(c.k, c.v, c.k_scale, c.v_scale)


# --------------------------------------------------------------------------- the plain forms

def _ancestors(parents: torch.Tensor, valid: torch.Tensor) -> torch.Tensor:
    """[B, n, n]: whether node j is node i or above it, from parents [B, n] (-1: none), by repeated squaring."""
    n = parents.shape[1]
    i = torch.arange(n, device=parents.device)
    up = (parents[:, :, None] == i) & valid[:, :, None] & valid[:, None, :]
    reach = ((i[:, None] == i) | up).float()
    for _ in range(max(1, (n - 1).bit_length())):
        reach = (torch.matmul(reach, reach) > 0).float()
    return reach > 0


def _padded(rows: torch.Tensor, cu: torch.Tensor, n: int):
    """Packed rows [T, ...] as [B, n, ...], and which of them are rows."""
    i = torch.arange(n, device=rows.device)
    valid = i < (cu[1:] - cu[:-1])[:, None]
    at = (cu[:-1, None].long() + i).clamp_max(len(rows) - 1)
    return rows[at], valid, at


def _plain_tables(s: dict) -> list:
    dev, bs, rows, table, free = s["table"].device, s["block"], s["rows"], s["table"], s["free"]
    length, new, held = s["seq_lens"].long(), s["new_lens"].long(), s["held"].long()
    ends = torch.cumsum(new, 0)
    total = (length + new + bs - 1) // bs
    fits = (new > 0) & (total <= table.shape[1]) & (ends <= rows)
    if s["nodes"]:
        fits &= new <= s["nodes"]
    need = torch.where(fits, (total - held).clamp_min(0), 0)
    last = torch.cumsum(need, 0)
    granted = fits & ((need == 0) | (s["taken"] + last <= len(free)))
    got = torch.where(granted, need, 0)
    first = s["taken"] + last - need
    i = torch.arange(table.shape[1], device=dev)
    fresh = (i >= held[:, None]) & (i < (held + got)[:, None])
    table = torch.where(fresh, free[(first[:, None] + i - held[:, None]).clamp(0, len(free) - 1)], table)
    r = torch.arange(rows, device=dev)
    seq = torch.searchsorted(ends, r, right=True).clamp_max(len(new) - 1)
    j = r - (ends - new)[seq]
    real = (r < ends[-1]) & granted[seq]
    at = length[seq] + j
    slots = table[seq, (at // bs).clamp_max(table.shape[1] - 1)].long() * bs + at % bs
    out = [(held + got).int(), (s["taken"] + got.sum()).int(),
           torch.where(new > 0, torch.where(granted, length + new, 0), length).int(),
           torch.cat([torch.zeros_like(ends[:1]), ends]).clamp_max(rows).int(), torch.where(real, slots, -1)]
    refused = ((new > 0) & ~granted).sum().int().view(1)
    if not s["nodes"]:
        return [table] + out + [torch.where(real, at, -1), refused]
    n = s["nodes"]
    parents, valid, _ = _padded(s["parents"], torch.cat([torch.zeros_like(ends[:1]), ends]), n)
    up = _ancestors(parents, valid)
    bits = 1 << torch.arange(64, device=dev)
    masks = (up.view(*up.shape[:2], n // 64, 64) * bits).sum(-1)  # bit 63 wraps to the sign
    depth = up.sum(-1) - 1
    k = j.clamp(0, n - 1)
    return [table] + out + [torch.where(real, length[seq] + depth[seq, k], -1), refused,
                            torch.where(real[:, None], masks[seq, k], 0)]


def _turned(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, inter: bool) -> torch.Tensor:
    half = cos.shape[-1]
    y = x.float()
    a, b = (y[..., 0:2 * half:2], y[..., 1:2 * half:2]) if inter else (y[..., :half], y[..., half:2 * half])
    u, v = a * cos - b * sin, b * cos + a * sin
    z = torch.stack([u, v], -1).flatten(-2) if inter else torch.cat([u, v], -1)
    return torch.cat([z, y[..., 2 * half:]], -1).to(x.dtype)


def _plain_rotary(s: dict) -> list:
    q, k = s["q"].detach(), s["k"].detach()
    angle = s["pos"].double()[:, None, None] * s["freq"]
    cos, sin = (torch.cos(angle) * s["scale"]).float(), (torch.sin(angle) * s["scale"]).float()
    out = [_turned(q, cos, sin, s["inter"]), _turned(k, cos, sin, s["inter"])]
    if "gq" in s:  # a rotation's transpose turns the other way
        out += [_turned(s["gq"], cos, -sin, s["inter"]), _turned(s["gk"], cos, -sin, s["inter"])]
    return out


def _values(x: torch.Tensor, scale) -> torch.Tensor:
    """Cache entries as 32-bit values; `scale` shaped like the blocks and heads of x."""
    if scale is None:
        return x.float()
    return x.view(torch.float8_e4m3fn).float() * scale.view(*scale.shape, *([1] * (x.dim() - scale.dim())))


def _plain_tree(s: dict) -> list:
    k, v, ks, vs = s["kv"]
    bs, n = s["block"], s["longest"]
    if "key" in s:
        blk, off = s["slots"] // bs, s["slots"] % bs
        k[blk, :, :, off] = s["key"].view(*s["key"].shape[:2], -1, k.shape[-1])
        v[blk, :, :, off] = s["value"]
    table = s["table"].long().clamp_min(0)
    b, m = table.shape
    hkv, d = v.shape[1], v.shape[2]
    kk = _values(k[table], None if ks is None else ks[table]).permute(0, 2, 1, 4, 3, 5).reshape(b, hkv, m * bs, d)
    vv = _values(v[table], None if vs is None else vs[table]).permute(0, 2, 1, 4, 3).reshape(b, hkv, m * bs, d)
    q, valid, at = _padded(s["q"], s["cu"], n)
    hq = q.shape[2]
    q = q.float().view(b, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    new = (s["cu"][1:] - s["cu"][:-1])[:, None]
    key = torch.arange(m * bs, device=q.device)
    j = key - (s["seq_lens"][:, None] - new)  # the key's node, below 0 in the context
    words = s["mask"][at].clone()
    bit = words.gather(2, (j.clamp(0, n - 1) // 64)[:, None, :].expand(-1, n, -1)) >> (j.clamp(0, n - 1) % 64)[:, None, :]
    seen = ((j < 0)[:, None, :] | ((bit & 1) > 0)) & (j < new)[:, None, :]
    x = torch.matmul(q, kk.transpose(2, 3)).view(b, hkv, hq // hkv, n, m * bs) * s["scale"]
    x = torch.where(seen[:, None, None], x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    y = torch.matmul(x.view(b, hkv, -1, m * bs), vv).view(b, hkv, hq // hkv, n, d).permute(0, 3, 1, 2, 4)
    out = torch.empty((len(s["q"]) + 1, hq, d), dtype=s["q"].dtype, device=q.device)
    out[torch.where(valid, at, len(s["q"]))] = y.reshape(b, n, hq, d).to(out.dtype)  # rows past a sequence's last go nowhere
    return [out[:-1]] + ([k, v] if "key" in s else [])


def _plain_accept(s: dict) -> list:
    n, p = s["longest"], s["depth"]
    parents, valid, at = _padded(s["parents"], s["cu"], n)
    draft, target = s["draft"][at], s["target"][at]
    i = torch.arange(n, device=at.device)
    match = valid & (parents >= 0) & (draft == target.gather(1, parents.long().clamp_min(0)))
    # of siblings that match, the first
    earlier = (parents[:, :, None] == parents[:, None, :]) & match[:, None, :] & (i[None, :] < i[:, None])
    match &= ~earlier.any(2)
    match[:, 0] = valid[:, 0]
    up = _ancestors(parents, valid)
    on = valid & ~(up & ~match[:, None, :]).any(2) & up[:, :, 0]
    depth = up.sum(2) - 1
    on &= depth < p
    path = torch.full((len(parents), p + 1), -1, dtype=torch.int32, device=at.device)
    path.scatter_(1, torch.where(on, depth, p), i.int().expand_as(on).contiguous())
    path = path[:, :p].contiguous()
    count = on.sum(1)
    last = path.gather(1, (count - 1)[:, None].clamp_min(0)).long()
    return [count.int(), path, target.gather(1, last)[:, 0], (s["seq_lens"] + count).int()]


def _pow2_scale(amax: torch.Tensor) -> torch.Tensor:
    """The smallest power of two at or above max(amax, 1e-10) / 448."""
    m, e = torch.frexp(amax.clamp_min(1e-10) / 448.0)
    return torch.ldexp(torch.ones_like(m), torch.where(m == 0.5, e - 1, e))


def _plain_compact(s: dict) -> list:
    k, v, ks, vs = s["kv"]
    bs, path = s["block"], s["path"].long()
    b, p = path.shape
    i = torch.arange(p, device=path.device)
    taken = i < s["accepted"][:, None]
    table, length = s["table"].long(), s["seq_lens"].long()[:, None]
    if ks is None:
        src = length + torch.where(taken, path, path[:, :1])  # what is not moved repeats the first
        dst = length + torch.where(taken, i, 0)
        seq = torch.arange(b, device=path.device)[:, None]
        sb, db = table[seq, src // bs], table[seq, dst // bs]
        kk, vv = k[sb, :, :, src % bs], v[sb, :, :, src % bs]
        k[db, :, :, dst % bs] = kk
        v[db, :, :, dst % bs] = vv
        return [k, v]
    # The tokens that change their place, block by block: what a block held before them is encoded
    # again where its scale grows; a block that they start is scaled by them alone.
    moved = taken & (path != i)
    start = length[:, 0] + torch.where(moved, i, p).amin(1)  # the first new place
    end = length[:, 0] + s["accepted"].long()
    start = torch.minimum(start, end)
    runs = torch.arange((p + bs - 2) // bs + 1, device=path.device)
    blk = start[:, None] // bs + runs
    use = (blk * bs < end[:, None])
    blk = torch.where(use, blk, start[:, None] // bs)  # a run too many repeats the first
    blk = torch.minimum(blk, ((end - 1).clamp_min(0) // bs)[:, None])
    ids = table.gather(1, blk)
    off = torch.arange(bs, device=path.device)
    pos = blk[:, :, None] * bs + off
    here = (pos >= start[:, None, None]) & (pos < end[:, None, None])
    first = (start[:, None] - blk * bs).clamp_min(0)
    node = path.gather(1, (pos - length[:, :, None]).clamp(0, p - 1).flatten(1)).view_as(pos).clamp_min(0)
    src = torch.where(here, length[:, :, None] + node, 0)
    sb = table.gather(1, (src // bs).flatten(1)).view_as(src)
    out = []
    for x, sc in ((k, ks), (v, vs)):
        old = x[ids]  # [B, R, H, ..., bs(, 16)]
        if x is k:
            old = old.permute(0, 1, 2, 3, 5, 4).flatten(3, 4)  # [B, R, H, D, bs]
            new = x[sb, :, :, src % bs].flatten(4)             # [B, R, bs, H, D]
        else:
            new = x[sb, :, :, src % bs]
        new = (new.contiguous().view(torch.float8_e4m3fn).float() * sc[sb][..., None]).permute(0, 1, 3, 4, 2)
        put = here[:, :, None, None, :]
        amax = torch.where(put, new.abs(), 0).amax((3, 4))
        held = sc[ids]
        want = torch.where(here.any(2)[:, :, None],
                           torch.where((first == 0)[:, :, None], _pow2_scale(amax), torch.maximum(held, _pow2_scale(amax))),
                           held)
        again = (old.contiguous().view(torch.float8_e4m3fn).float() * (held / want)[..., None, None])
        before = (off < first[:, :, None])[:, :, None, None, :] & (want > held)[..., None, None]
        code = lambda y: y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)  # noqa: E731
        old = torch.where(before, code(again), old)
        old = torch.where(put, code(new / want[..., None, None]), old)
        if x is k:
            old = old.unflatten(3, (-1, 16)).permute(0, 1, 2, 3, 5, 4)
        out.append((x, sc, old, want))
    for x, sc, old, want in out:
        x[ids] = old
        sc[ids] = want
    return _contents(k, v, ks, vs)


_PLAIN = {"tables": _plain_tables, "rotary": _plain_rotary, "tree": _plain_tree, "accept": _plain_accept,
          "compact": _plain_compact}


def run(s: dict) -> list:
    return _run_own(s) if own else _PLAIN[s["kind"]](s)


# --------------------------------------------------------------------------- the results in float64

def _turn64(x, pos, freq, scale, inter, way):
    x = x.detach().double()
    half = len(freq)
    a = pos.double()[:, None] * freq
    z = torch.polar(torch.full_like(a, scale), way * a)[:, None, :]
    first = torch.arange(half, device=x.device) * (2 if inter else 1)
    second = first + (1 if inter else half)
    y = x.clone()
    w = torch.complex(x[:, :, first].contiguous(), x[:, :, second].contiguous()) * z
    y[:, :, first], y[:, :, second] = w.real, w.imag
    return y


def exact(case: dict, seed: int):
    kind = case["kind"]
    if kind == "rotary":
        x = _rotary_inputs(case, seed)
        f = (x["pos"], x["freq"], x["scale"], case["inter"])
        out = [_turn64(x["q"], *f, 1), _turn64(x["k"], *f, 1)]
        return out + ([_turn64(x["gq"], *f, -1), _turn64(x["gk"], *f, -1)] if case["grad"] else [])
    if kind == "tree":
        hq, hkv, d = MODELS[case["model"]]
        g = hq // hkv
        x = _tree_inputs(case, seed)
        k, v, ks, vs = x["kv"]
        if "key" in x:
            blk, off = x["slots"] // case["block"], x["slots"] % case["block"]
            for t in range(hkv):
                k[blk, t, :, off] = x["key"][:, t].view(len(blk), -1, k.shape[-1])
                v[blk, t, :, off] = x["value"][:, t]
        out = torch.zeros(x["q"].shape, dtype=torch.float64, device=_device())
        cu, lens = x["cu"].tolist(), x["seq_lens"].tolist()
        for i, n in enumerate(lens):
            m = cu[i + 1] - cu[i]
            ids = x["table"][i, :-(-n // case["block"])].long()
            bits = [x["mask"][cu[i]:cu[i + 1], j // 64] >> (j % 64) & 1 for j in range(m)]
            seen = torch.ones((m, n), dtype=torch.bool, device=_device())
            seen[:, n - m:] = torch.stack(bits, 1) > 0
            for t in range(hkv):
                kk, vv = k[ids, t], v[ids, t]
                if ks is not None:
                    kk = kk.view(torch.float8_e4m3fn).double() * ks[ids, t].double()[:, None, None, None]
                    vv = vv.view(torch.float8_e4m3fn).double() * vs[ids, t].double()[:, None, None]
                kk = kk.double().transpose(1, 2).reshape(-1, d)[:n]
                vv = vv.double().transpose(1, 2).reshape(-1, d)[:n]
                q = x["q"][cu[i]:cu[i + 1], t * g:(t + 1) * g].double().transpose(0, 1).reshape(-1, d)
                a = (q @ kk.T.contiguous() * d ** -0.5).view(g, m, n).masked_fill_(~seen, -math.inf)
                out[cu[i]:cu[i + 1], t * g:(t + 1) * g] = (torch.softmax(a, -1).view(-1, n) @ vv).view(g, m, d).transpose(0, 1)
        return [out] + ([None, None] if "key" in x else [])
    if kind == "compact" and case["kv"] == "bf16":
        x = _compact_inputs(case, seed)
        k, v = x["kv"][0].double().cpu(), x["kv"][1].double().cpu()
        bs = case["block"]
        for row, n, p, a in zip(x["table"].tolist(), x["seq_lens"].tolist(), x["path"].tolist(), x["accepted"].tolist()):
            at = lambda i: (row[(n + i) // bs], (n + i) % bs)  # noqa: E731
            rows = [(k[at(p[i])[0], :, :, at(p[i])[1]].clone(), v[at(p[i])[0], :, :, at(p[i])[1]].clone()) for i in range(a)]
            for i, (kk, vv) in enumerate(rows):
                k[at(i)[0], :, :, at(i)[1]], v[at(i)[0], :, :, at(i)[1]] = kk, vv
        return [k, v]
    return None  # whole numbers, and 8-bit values at their scales, which the documented rule fixes
