"""What a step of drafted tokens costs an fp8 cache in accuracy, next to the same tokens appended one by one (CPU,
on the oracle, whose caches are the GPU's bit for bit).

Bounds. A code is within half a step of the value: 2^-4 of its magnitude, or 2^-10 of the block's scale
where e4m3 is subnormal. Re-encoding at a grown scale is exact but for subnormals, half a step of the grown scale each
time; scales are powers of two, so these halves sum to less than twice the last one. A token appended
once is thus within 2^-4 |x| + 2 * 2^-10 S of x, S the largest scale its block has had; one that is then moved
adds as much again for its second code, of a value up to 2^-4 |x| + 2^-9 S' larger, in a block of scales up to S.
"""

import numpy as np
import pytest

from oracle import fp8, paged, tree

BS, H, D, CTX, NODES = 16, 2, 64, 21, 24


def _values(k, v, ks, vs):
    kl = np.ascontiguousarray(paged.k_logical(k)).reshape(len(k), BS, H, D)
    return [fp8.dequantize(x, s[:, None, :, None]) for x, s in ((kl, ks), (paged.v_logical(v), vs))]


@pytest.mark.parametrize("seed", range(3))
@pytest.mark.parametrize("loud", [1.0, 300.0])  # magnitude of the rejected tokens
def test_drafted_tokens_next_to_tokens_one_by_one(seed, loud):
    rng = np.random.default_rng(seed)
    table = np.array([[3, 1, 4]])
    path = np.array([0, *np.sort(rng.choice(np.arange(1, NODES), 7, replace=False))])
    x = [paged.f32_to_bf16(rng.normal(size=(CTX + NODES, H, D)).astype(np.float32)) for _ in range(2)]
    rejected = CTX + np.setdiff1d(np.arange(NODES), path)
    for y in x:
        y[rejected] = paged.f32_to_bf16(paged.bf16_to_f32(y[rejected]) * np.float32(loud))
    slot = lambda p: table[0, p // BS] * BS + p % BS  # noqa: E731

    def cache():
        c = [*paged.empty_cache(6, BS, H, D, dtype=np.uint8), *(np.zeros((6, H), np.float32) for _ in range(2))]
        paged.append_fp8(*c, x[0][:CTX], x[1][:CTX], slot(np.arange(CTX)))
        return c

    one, drafted = cache(), cache()
    kept = CTX + path
    largest = np.maximum(one[2], one[3])
    for j, p in enumerate(kept):
        paged.append_fp8(*one, x[0][p:p + 1], x[1][p:p + 1], slot(np.array([CTX + j])))
    nodes = np.arange(CTX, CTX + NODES)
    paged.append_fp8(*drafted, x[0][nodes], x[1][nodes], slot(nodes))
    for s in (*one[2:], *drafted[2:]):
        largest = np.maximum(largest, s)
    grown = [s.copy() for s in drafted[2:]]
    tree.compact(*drafted, table, np.array([CTX]), path[None].astype(np.int32), np.array([len(path)]))
    at = slot(CTX + np.arange(len(path)))
    S = largest.max(axis=0)[None, :, None]  # of any block, per head
    errors = []
    for got, ref, bits in zip(_values(*drafted), _values(*one), x):
        want = paged.bf16_to_f32(bits[kept]).astype(np.float64)
        first = np.abs(want) / 16 + 2 * S / 1024
        assert (np.abs(ref[at // BS, at % BS] - want) <= first).all()
        err = np.abs(got[at // BS, at % BS] - want)
        assert (err <= first + (np.abs(want) + first) / 16 + 2 * S / 1024).all()
        errors.append((np.sqrt((err ** 2).mean()), np.sqrt(((ref[at // BS, at % BS] - want) ** 2).mean())))
    if loud > 1:  # the block that holds the context's end keeps the scale that the rejected tokens gave it
        block = table[0, CTX // BS]
        assert all((s[block] > o[block]).all() for s, o in zip(grown, one[2:]))
        assert all((d[block] == s[block]).all() for d, s in zip(drafted[2:], grown))
        assert all(e > o for e, o in errors)
