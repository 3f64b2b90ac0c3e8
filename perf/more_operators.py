"""The measured calls between a layer's projections and its attention: norms, rotary positions, the append.

``norm_rotary`` takes the queries and keys of a fused projection, norms every head (root mean square, with
the weights that queries and keys have of their own) and turns it by its token's position, with gradients
of the heads and of the weights for training. ``apply_rotary`` with ``axes`` turns heads by positions that
have several axes (time, height and width of images and video). ``rotary_append`` does the norm and the
rotation on the way: queries to the attention, keys and values into the paged cache, bf16 or fp8.
``mla_rotary_append`` is the same for a latent cache: the compressed entry normed, the shared key turned.

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

EPS = 1e-6


def listed() -> list[dict]:
    return [
        # The heads of one new token, normed and turned: a decode step's latency.
        dict(name="norm_token", kind="norm", model="qwen3-4b", tokens=1, rotary=128, inter=False, dtype="bf16",
             weights="head_dim", axes=0, mixed=False, top=32768, base=1e6, grad=False),
        # The prompts of a step, outside a cache (scoring, the forward pass of training).
        dict(name="norm_prompts", kind="norm", model="qwen3-4b", tokens=16384, rotary=128, inter=False, dtype="bf16",
             weights="head_dim", axes=0, mixed=False, top=32768, base=1e6, grad=False),
        # A training batch of odd size, forward and backward, with the weights' gradients.
        dict(name="norm_train", kind="norm", model="qwen3-0.6b", tokens=8191, rotary=128, inter=False, dtype="bf16",
             weights="head_dim", axes=0, mixed=False, top=32768, base=1e6, grad=True),
        # A short float32 fine-tuning batch whose heads have weights of their own, half of each turned, pairs adjacent.
        dict(name="norm_train_heads", kind="norm", model="qwen2.5-7b", tokens=601, rotary=64, inter=True,
             dtype="fp32", weights="each_head", axes=0, mixed=False, top=4096, base=1e4, grad=True),
        # Images in a prompt: positions of three axes, each its own run of a head's pairs.
        dict(name="axes_images", kind="axes", model="qwen2.5-7b", tokens=12289, rotary=128, inter=False, dtype="bf16",
             axes=3, mixed=False, top=32768, base=1e6, grad=False),
        # The patches of one small image in training: two axes that take turns over the pairs.
        dict(name="axes_train", kind="axes", model="qwen3-0.6b", tokens=1023, rotary=128, inter=False, dtype="fp16",
             axes=2, mixed=True, top=64, base=1e4, grad=True),
        # The decode step of a rollout batch: one token of each of 64 sequences.
        dict(name="append_decode", kind="append", model="qwen3-4b", kv="bf16", batch=64, ctx_lo=65, ctx_hi=500,
             new_lo=1, new_hi=1, block=16, norm=True, rotary=128, inter=False, axes=0, mixed=False, base=1e6),
        # Eight prompts of 2,048 tokens.
        dict(name="append_prompts", kind="append", model="qwen3-4b", kv="bf16", batch=8, ctx_lo=0, ctx_hi=0,
             new_lo=2048, new_hi=2048, block=16, norm=True, rotary=128, inter=False, axes=0, mixed=False, base=1e6),
        # Ragged prompt chunks behind ragged contexts, fp8 KV, heads turned without a norm.
        dict(name="append_chunks_fp8", kind="append", model="qwen2.5-7b", kv="fp8_e4m3", batch=7, ctx_lo=5,
             ctx_hi=403, new_lo=333, new_hi=2047, block=16, norm=False, rotary=128, inter=False, axes=0, mixed=False,
             base=1e6),
        # A few sequences of a small model, one token each, fp8 KV in larger blocks.
        dict(name="append_few_fp8", kind="append", model="qwen2.5-0.5b", kv="fp8_e4m3", batch=5, ctx_lo=40,
             ctx_hi=333, new_lo=1, new_hi=1, block=32, norm=True, rotary=64, inter=False, axes=0, mixed=False, base=1e6),
        # The latent entries of a decode step of 32 sequences, 128 query heads.
        dict(name="latent_decode", kind="latent", heads=128, rank=512, rope=64, batch=32, ctx_lo=65, ctx_hi=500,
             new_lo=1, new_hi=1, block=64, norm=True, inter=True, base=1e4),
        # Ragged prompts into a latent cache.
        dict(name="latent_prompts", kind="latent", heads=128, rank=512, rope=64, batch=4, ctx_lo=0, ctx_hi=77,
             new_lo=301, new_hi=2047, block=64, norm=True, inter=True, base=1e4),
    ]


_MAX_VALUES = 16384 * 40 * 128  # head values of the largest drawn pass


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _range(rng, lo: int, hi: int) -> tuple[int, int]:
    top = _log_int(rng, lo, hi)
    return rng.choice([top, max(lo, top // 3), lo]), top


def draw(rng) -> dict:
    kind = rng.choice(["norm", "norm", "norm", "axes", "axes", "append", "append", "append", "latent"])
    if kind in ("norm", "axes"):
        model = rng.choice(sorted(MODELS))
        hq, hkv, d = MODELS[model]
        grad = bool(rng.random() < 0.5)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        cost = (hq + hkv) * d * (2.5 if grad else 1) * (2 if dtype == "fp32" else 1)
        axes = rng.choice([2, 3]) if kind == "axes" else rng.choice([0, 0, 3])
        case = dict(kind=kind, model=model, tokens=_log_int(rng, 1, max(1, int(_MAX_VALUES / cost))),
                    rotary=rng.choice([d, d, d // 2, 2 * rng.randint(4, d // 2)]), inter=bool(rng.random() < 0.4),
                    dtype=dtype, axes=axes, mixed=bool(rng.random() < 0.5), top=_log_int(rng, 64, 1 << 18),
                    base=rng.choice([1e4, 1e6]), grad=grad)
        if kind == "norm":
            case["weights"] = rng.choice(["head_dim", "head_dim", "head_dim", "each_head", "none"])
        return case
    c_lo, c_hi = rng.choice([(0, 0), _range(rng, 1, 600), _range(rng, 1, 600)])
    n_lo, n_hi = rng.choice([(1, 1), _range(rng, 1, 2048)])
    case = dict(kind=kind, batch=_log_int(rng, 1, 256), ctx_lo=c_lo, ctx_hi=c_hi, new_lo=n_lo, new_hi=n_hi,
                norm=bool(rng.random() < 0.7), base=rng.choice([1e4, 1e6]))
    if kind == "append":
        model = rng.choice(sorted(MODELS))
        hq, hkv, d = MODELS[model]
        case.update(model=model, kv=rng.choice(["bf16", "fp8_e4m3"]), block=rng.choice([16, 16, 32, 64]),
                    rotary=rng.choice([d, d, d // 2]), inter=bool(rng.random() < 0.3), axes=rng.choice([0, 0, 0, 3]),
                    mixed=bool(rng.random() < 0.5))
        row = (hq + 2 * hkv) * d
    else:
        case.update(heads=rng.choice([16, 64, 128]), rank=512, rope=64, block=rng.choice([16, 64]),
                    inter=bool(rng.random() < 0.7))
        row = case["heads"] * 64 + 576
    while case["batch"] * n_hi * row > _MAX_VALUES or case["batch"] * (c_hi + n_hi) > 1 << 17:
        case["batch"] = max(1, case["batch"] // 2)
    return case


# --------------------------------------------------------------------------- sizes

def _spread(lo: int, hi: int, n: int) -> list[int]:
    """n lengths spread evenly over [lo, hi]: the same for every seed (which sequence has which is not)."""
    return [lo + (hi - lo) * i // (n - 1) if n > 1 else hi for i in range(n)]


def _lens(case: dict) -> tuple[list[int], list[int]]:
    """Context and new lengths; the new ones run the other way."""
    return _spread(case["ctx_lo"], case["ctx_hi"], case["batch"]), _spread(case["new_lo"], case["new_hi"], case["batch"])[::-1]


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind in ("norm", "axes"):
        hq, hkv, d = MODELS[case["model"]]
        esz = 4 if case["dtype"] == "fp32" else 2
        values = case["tokens"] * (hq + hkv) * d * (2 if case["grad"] else 1)
        turned = values * case["rotary"] // d
        norm = (4 * values * (2 if case["grad"] else 1)) if kind == "norm" else 0
        return {"bytes": 2 * values * esz + case["tokens"] * 8 * max(1, case["axes"]), "flops": 3 * turned + norm}
    _, new = _lens(case)
    t = sum(new)
    if kind == "append":
        hq, hkv, d = MODELS[case["model"]]
        esz = 2 if case["kv"] == "bf16" else 1
        return {"bytes": t * (4 * hq * d + 2 * hkv * d * (2 + esz) + 8 + 8 * max(1, case["axes"])),
                "flops": t * (hq + hkv) * (3 * case["rotary"] + (4 * d if case["norm"] else 0))}
    width = case["rank"] + case["rope"]
    return {"bytes": t * (4 * case["heads"] * case["rope"] + 4 * width + 16),
            "flops": t * ((case["heads"] + 1) * 3 * case["rope"] + (4 * case["rank"] if case["norm"] else 0))}


# --------------------------------------------------------------------------- inputs

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _device() -> torch.device:
    return torch.device("cuda", torch.cuda.current_device())


def _gens(seed: int):
    g = torch.Generator(device=_device())
    g.manual_seed(seed)
    h = torch.Generator()
    h.manual_seed(seed)
    return g, h


def _normal(gen, shape, dtype=torch.bfloat16) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype, device=_device()).normal_(generator=gen)


def _weight(gen, shape, dtype) -> torch.Tensor:
    return (1 + 0.25 * _normal(gen, shape, torch.float32)).to(dtype)


def _axis_of_pair(half: int, n: int, mixed: bool) -> torch.Tensor:
    """The axis of every pair: of each axis its run of pairs, or the axes in turn (what is left is the first's)."""
    others = 3 * half // 8 if n == 3 else half // 2
    sections = [half - (n - 1) * others] + [others] * (n - 1)
    if not mixed:
        return torch.repeat_interleave(torch.arange(n), torch.tensor(sections)).int().to(_device())
    i = torch.arange(half)
    return torch.where(i < n * min(others, half // n), i % n, 0).int().to(_device())


def _grid_positions(start: int, tokens: int, axes: int, top: int) -> torch.Tensor:
    """[axes, tokens]: text, whose axes agree, and behind it images of 24 x 24 patches, one after the other in time."""
    i = torch.arange(tokens, device=_device())
    text = tokens // 4
    j = (i - text).clamp_min(0)
    per = [j // 576, j // 24 % 24, j % 24][-axes:]
    pos = torch.stack([torch.where(i < text, i, text + p) for p in per])
    return (start + pos) % top


def _rotary(case: dict, tokens: int, start: int, top: int) -> dict:
    r = case["rotary"] if "rotary" in case else case["rope"]
    freq = case["base"] ** (-torch.arange(0, r, 2, dtype=torch.float64, device=_device()) / r)
    n = case.get("axes", 0)
    if not n:
        return dict(freq=freq, axes=None, pos=(start + torch.arange(tokens, device=_device())) % top)
    return dict(freq=freq, axes=_axis_of_pair(r // 2, n, case["mixed"]), pos=_grid_positions(start, tokens, n, top))


def _rows_inputs(case: dict, seed: int) -> dict:
    gen, h = _gens(seed)
    hq, hkv, d = MODELS[case["model"]]
    t, dt = case["tokens"], _DTYPES[case["dtype"]]
    start = int(torch.randint(0, case["top"], (1,), generator=h))
    # q, k and v lie side by side, as a fused projection leaves them; heads differ in size
    x = _normal(gen, (t, hq + 2 * hkv, d), dt)
    x *= torch.exp(_normal(gen, (1, hq + 2 * hkv, 1), torch.float32)).to(dt)
    out = dict(q=x[:, :hq], k=x[:, hq:hq + hkv], **_rotary(case, t, start, case["top"]))
    if case["grad"]:
        out.update(gq=_normal(gen, (t, hq, d), dt), gk=_normal(gen, (t, hkv, d), dt))
    if case["kind"] == "norm":
        each = case["weights"] == "each_head"
        for name, n in (("qw", hq), ("kw", hkv)):
            out[name] = None if case["weights"] == "none" else _weight(gen, (n, d) if each else (d,), dt)
    return out


def _sequences(case: dict, h) -> dict:
    """Slots and positions of the new tokens of sequences whose blocks are dealt from a shuffled pool."""
    ctx, new = _lens(case)
    order = torch.randperm(len(ctx), generator=h).tolist()
    ctx, new, bs = [ctx[i] for i in order], [new[i] for i in order], case["block"]
    need = [-(-(c + n) // bs) for c, n in zip(ctx, new)]
    perm = torch.randperm(sum(need), generator=h)
    slots, pos, at = [], [], 0
    for c, n, m in zip(ctx, new, need):
        p = torch.arange(c, c + n)
        slots.append(perm[at:at + m][p // bs] * bs + p % bs)
        pos.append(p)
        at += m
    return dict(slots=torch.cat(slots).to(_device()), at=torch.cat(pos).to(_device()), blocks=sum(need), block=bs)


def _append_inputs(case: dict, seed: int) -> dict:
    gen, h = _gens(seed)
    hq, hkv, d = MODELS[case["model"]]
    s = _sequences(case, h)
    t, bs, blocks = len(s["slots"]), s["block"], s["blocks"]
    x = _normal(gen, (t, hq + 2 * hkv, d))
    x *= torch.exp(_normal(gen, (1, hq + 2 * hkv, 1), torch.float32)).bfloat16()
    s.update(q=x[:, :hq], key=x[:, hq:hq + hkv], value=x[:, hq + hkv:], **_rotary(case, t, 0, 1 << 30))
    if not case["axes"]:
        s["pos"] = s["at"]
    s.update(qw=_weight(gen, (d,), x.dtype) if case["norm"] else None,
             kw=_weight(gen, (d,), x.dtype) if case["norm"] else None)
    # one layer's cache in the library's documented layout: K [N, H, D/x, B, x], V [N, H, D, B], scales
    if case["kv"] == "bf16":
        s["kv"] = [_normal(gen, (blocks, hkv, d // 8, bs, 8)), _normal(gen, (blocks, hkv, d, bs)), None, None]
    else:
        kv = []
        for shape in ((blocks, hkv, d // 16, bs, 16), (blocks, hkv, d, bs)):
            sc = torch.ldexp(torch.ones((blocks, hkv), device=_device()),
                             torch.randint(-8, -4, (blocks, hkv), generator=gen, device=_device()))
            y = _normal(gen, shape, torch.float32) / sc.view(blocks, hkv, *([1] * (len(shape) - 2)))
            kv.append((y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), sc))
        s["kv"] = [kv[0][0], kv[1][0], kv[0][1], kv[1][1]]
    return s


def _latent_inputs(case: dict, seed: int) -> dict:
    gen, h = _gens(seed)
    s = _sequences(case, h)
    t, heads, rank, rope = len(s["slots"]), case["heads"], case["rank"], case["rope"]
    # q_pe is the end of every query head's projection; kv_c and k_pe lie side by side
    q, kv = _normal(gen, (t, heads, 128 + rope)), _normal(gen, (t, rank + rope))
    kv *= 3
    s.update(_rotary(case, t, 0, 1 << 30))
    s.update(q=q[:, :, 128:], kv_c=kv[:, :rank], k_pe=kv[:, rank:], pos=s["at"],
             kw=_weight(gen, (rank,), q.dtype) if case["norm"] else None,
             latent=_normal(gen, (s["blocks"], s["block"], rank + rope)))
    return s


_INPUTS = {"norm": _rows_inputs, "axes": _rows_inputs, "append": _append_inputs, "latent": _latent_inputs}


def prepare(case: dict, seed: int) -> dict:
    s = _INPUTS[case["kind"]](case, seed)
    s.update(kind=case["kind"], inter=case["inter"], norm=case.get("norm", True), fp8=case.get("kv") == "fp8_e4m3")
    if case.get("grad"):
        for name in ("q", "k", "qw", "kw"):
            if s.get(name) is not None:
                s[name] = s[name].detach().requires_grad_(True)
    if own and "kv" in s:  # the layer's cache, which a serving program keeps
        from wavelet_amd import PagedKVCache

        _, hkv, d = MODELS[case["model"]]
        c = s["cache"] = PagedKVCache(s["blocks"], s["block"], hkv, d, kv_dtype=case["kv"], device=_device())
        for name, x in zip(("k", "v", "k_scale", "v_scale"), s.pop("kv")):
            if x is not None:
                getattr(c, name).copy_(x)
    if own and "latent" in s:
        from wavelet_amd import MLALatentCache

        c = s["cache"] = MLALatentCache(s["blocks"], s["block"], case["rank"], case["rope"], device=_device())
        c.latent.copy_(s.pop("latent"))
    return s


# --------------------------------------------------------------------------- the framework's calls

def _contents(k, v, ks, vs) -> list:
    """A cache as the values that it holds: bf16 tensors, or fp8 values with their blocks' scales."""
    return [k, v] if ks is None else [k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), ks, vs]


def _run_own(s: dict) -> list:
    import wavelet_amd as w

    if s["kind"] == "append":
        c = s["cache"]
        q = w.rotary_append(s["q"], s["key"], s["value"], c, s["slots"], s["pos"], s["freq"], q_weight=s["qw"],
                            k_weight=s["kw"], eps=EPS if s["norm"] else None, axes=s["axes"], interleaved=s["inter"])
        return [q] + _contents(c.k, c.v, c.k_scale, c.v_scale)
    if s["kind"] == "latent":
        q = w.mla_rotary_append(s["q"], s["kv_c"], s["k_pe"], s["cache"], s["slots"], s["pos"], s["freq"],
                                kv_weight=s["kw"], eps=EPS if s["norm"] else None, interleaved=s["inter"])
        return [q, s["cache"].latent]
    if s["kind"] == "axes":
        q, k = w.apply_rotary(s["q"], s["k"], s["pos"], s["freq"], axes=s["axes"], interleaved=s["inter"])
    else:
        q, k = w.norm_rotary(s["q"], s["k"], s["pos"], s["freq"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                             axes=s["axes"], interleaved=s["inter"])
    if "gq" not in s:
        return [q, k]
    leaves = [x for x in (s["q"], s["k"], s.get("qw"), s.get("kw")) if x is not None]
    return [q.detach(), k.detach(), *torch.autograd.grad([q, k], leaves, [s["gq"], s["gk"]])]


# --------------------------------------------------------------------------- the plain forms

def _angles(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """Cosines and sines [T, 1, pairs] in 32 bits, of angles taken in 64."""
    pos = s["pos"][:, None] if s["axes"] is None else s["pos"][s["axes"].long()].T
    angle = (pos.double() * s["freq"])[:, None]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _turned(y: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, inter: bool) -> torch.Tensor:
    half = cos.shape[-1]
    a, b = (y[..., 0:2 * half:2], y[..., 1:2 * half:2]) if inter else (y[..., :half], y[..., half:2 * half])
    u, v = a * cos - b * sin, b * cos + a * sin
    z = torch.stack([u, v], -1).flatten(-2) if inter else torch.cat([u, v], -1)
    return torch.cat([z, y[..., 2 * half:]], -1)


def _normed(x: torch.Tensor, weight) -> torch.Tensor:
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return y if weight is None else y * weight.float()


def _plain_rows(s: dict) -> list:
    cos, sin = _angles(s)
    norm = s["kind"] == "norm"
    out, grads, weights = [], [], []
    for x, w, g in ((s["q"], s.get("qw"), s.get("gq")), (s["k"], s.get("kw"), s.get("gk"))):
        x, w = x.detach(), None if w is None else w.detach()
        y = x.float()
        out.append(_turned(_normed(y, w) if norm else y, cos, sin, s["inter"]).to(x.dtype))
        if g is None:
            continue
        z = _turned(g.float(), cos, -sin, s["inter"])  # a rotation's transpose turns the other way
        if norm:
            r = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
            if w is not None:
                dw = z * y * r
                weights.append(dw.sum((0, 1) if w.dim() == 1 else 0).to(x.dtype))
                z = z * w.float()
            z = r * (z - y * r * r * (z * y).mean(-1, keepdim=True))
        grads.append(z.to(x.dtype))
    return out + grads + weights


def _pow2_scale(amax: torch.Tensor) -> torch.Tensor:
    """The smallest power of two at or above max(amax, 1e-10) / 448."""
    m, e = torch.frexp(amax.clamp_min(1e-10) / 448.0)
    return torch.ldexp(torch.ones_like(m), torch.where(m == 0.5, e - 1, e))


def _plain_append(s: dict) -> list:
    cos, sin = _angles(s)
    q, key, value = s["q"].float(), s["key"].float(), s["value"]
    if s["norm"]:
        q, key = _normed(q, s["qw"]), _normed(key, s["kw"])
    q, key = (_turned(x, cos, sin, s["inter"]).bfloat16() for x in (q, key))
    k, v, ks, vs = s["kv"]
    bs = s["block"]
    blk, off = s["slots"] // bs, s["slots"] % bs
    if ks is None:
        k[blk, :, :, off] = key.view(*key.shape[:2], -1, k.shape[-1])
        v[blk, :, :, off] = value
        return [q, k, v]
    # A block's new tokens are one run: a run that begins the block scales it alone, otherwise its
    # scale can only grow, and what the block held is coded again at the grown one.
    n, hkv = len(k), k.shape[1]
    first = torch.full((n,), bs, device=blk.device).scatter_reduce(0, blk, off, "amin")
    used = first < bs
    code = lambda x: x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)  # noqa: E731
    for x, sc, new in ((k, ks, key.float()), (v, vs, value.float())):
        amax = torch.zeros((n, hkv), device=blk.device).scatter_reduce(
            0, blk[:, None].expand(-1, hkv), new.abs().amax(-1), "amax")
        want = torch.where((first == 0)[:, None], _pow2_scale(amax), torch.maximum(sc, _pow2_scale(amax)))
        want = torch.where(used[:, None], want, sc)
        tail = [1] * (x.dim() - 2)
        again = code(x.view(torch.float8_e4m3fn).float() * (sc / want).view(n, hkv, *tail))
        slot = torch.arange(bs, device=blk.device).view([bs, 1] if x is k else [bs])
        before = (slot < first.view(n, *([1] * (x.dim() - 1)))) & (want > sc).view(n, hkv, *tail)
        x.copy_(torch.where(before, again, x))
        new = code(new / want[blk][..., None])
        x[blk, :, :, off] = new.view(*new.shape[:2], -1, 16) if x is k else new
        sc.copy_(want)
    return [q] + _contents(k, v, ks, vs)


def _plain_latent(s: dict) -> list:
    cos, sin = _angles(s)
    c = s["kv_c"].float()
    if s["norm"]:
        c = _normed(c, s["kw"])
    pe = _turned(s["k_pe"].float()[:, None], cos, sin, s["inter"])[:, 0]
    s["latent"].view(-1, s["latent"].shape[-1])[s["slots"]] = torch.cat([c, pe], -1).bfloat16()
    return [_turned(s["q"].float(), cos, sin, s["inter"]).bfloat16(), s["latent"]]


_PLAIN = {"norm": _plain_rows, "axes": _plain_rows, "append": _plain_append, "latent": _plain_latent}


def run(s: dict) -> list:
    return _run_own(s) if own else _PLAIN[s["kind"]](s)


# --------------------------------------------------------------------------- the results in float64

def _phase64(x: dict, way: int) -> torch.Tensor:
    """e^(i angle) [T, pairs]."""
    if x["axes"] is None:
        a = torch.outer(x["pos"].double(), x["freq"])
    else:
        a = torch.stack([x["pos"][ax].double() * f for ax, f in zip(x["axes"].tolist(), x["freq"])], 1)
    return torch.polar(torch.ones_like(a), way * a)


def _turn64(y: torch.Tensor, z: torch.Tensor, inter: bool) -> torch.Tensor:
    half = z.shape[1]
    first = torch.arange(half, device=y.device) * (2 if inter else 1)
    second = first + (1 if inter else half)
    out = y.clone()
    w = torch.complex(y[:, :, first].contiguous(), y[:, :, second].contiguous()) * z[:, None]
    out[:, :, first], out[:, :, second] = w.real, w.imag
    return out


def _unit64(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x over its root mean square, and that."""
    rms = (torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / x.shape[-1] + EPS).sqrt()
    return x / rms, rms


def exact(case: dict, seed: int):
    kind = case["kind"]
    x = _INPUTS[kind](case, seed)
    z, inter = _phase64(x, 1), case["inter"]
    if kind in ("norm", "axes"):
        out, grads, weights = [], [], []
        for name in ("q", "k"):
            v = x[name].double()
            w = x.get(name + "w")
            w64 = 1.0 if w is None else w.double()
            unit, rms = _unit64(v) if kind == "norm" else (v, 1.0)
            out.append(_turn64(unit * w64, z, inter))
            if case["grad"]:
                back = _turn64(x["g" + name].double(), z.conj(), inter)
                if w is not None:
                    weights.append((back * unit).sum(0) if w.dim() == 2 else (back * unit).sum(0).sum(0))
                if kind == "norm":
                    back = back * w64
                    back = (back - unit * ((back * unit).sum(-1, keepdim=True) / v.shape[-1])) / rms
                grads.append(back)
        return out + grads + weights
    if kind == "latent":
        c = x["kv_c"].double()
        if case["norm"]:
            c = _unit64(c)[0] * x["kw"].double()
        latent = x["latent"].double()
        bs = case["block"]
        latent[x["slots"] // bs, x["slots"] % bs, :case["rank"]] = c
        latent[x["slots"] // bs, x["slots"] % bs, case["rank"]:] = _turn64(x["k_pe"].double()[:, None], z, inter)[:, 0]
        return [_turn64(x["q"].double(), z, inter), latent]
    q, key, value = x["q"].double(), x["key"].double(), x["value"].double()
    if case["norm"]:
        q, key = _unit64(q)[0] * x["qw"].double(), _unit64(key)[0] * x["kw"].double()
    q, key = _turn64(q, z, inter), _turn64(key, z, inter)
    k, v, ks, vs = x["kv"]
    bs, (_, hkv, d) = case["block"], MODELS[case["model"]]
    slots = x["slots"].tolist()
    if ks is None:
        k, v = k.double(), v.double()
        for h in range(hkv):
            blk, off = x["slots"] // bs, x["slots"] % bs
            k[blk, h, :, off] = key[:, h].reshape(len(slots), -1, 8)
            v[blk, h, :, off] = value[:, h]
        return [q, k, v]
    # the cache holds what it codes as bf16 keys and values at a power-of-two scale, run by run
    key = key.bfloat16().double()
    k, v = (y.view(torch.float8_e4m3fn).double() for y in (k, v))
    ks, vs = ks.double(), vs.double()

    def coded(y):
        return y.clamp(-448, 448).float().to(torch.float8_e4m3fn).double()  # (bf16 values over powers of two: exact)

    i = 0
    while i < len(slots):
        b, j = slots[i] // bs, i
        while j < len(slots) and slots[j] // bs == b:
            j += 1
        o, n = slots[i] % bs, j - i
        for y, sc, new in ((k, ks, key[i:j]), (v, vs, value[i:j])):
            step = torch.exp2(torch.ceil(torch.log2((new.abs().amax((0, 2)).clamp_min(1e-10) / 448))))
            held = sc[b].clone()
            want = step if o == 0 else torch.maximum(held, step)
            scaled = coded(new / want[None, :, None])
            if o > 0:
                ratio = (held / want).view(hkv, 1, 1)
                if y is k:
                    y[b, :, :, :o] = coded(y[b, :, :, :o] * ratio[..., None])
                else:
                    y[b, :, :, :o] = coded(y[b, :, :, :o] * ratio)
            if y is k:
                y[b, :, :, o:o + n] = scaled.view(n, hkv, d // 16, 16).permute(1, 2, 0, 3)
            else:
                y[b, :, :, o:o + n] = scaled.permute(1, 2, 0)
            sc[b] = want
        i = j
    return [q, k, v, ks, vs]
