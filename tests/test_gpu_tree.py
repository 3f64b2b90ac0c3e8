"""Attention of drafted tokens over the paged cache on the GPU, against the float64 oracle.

Tolerance as for decode and prefill (kvcase.check_attention): |got - ref| <= 2e-2 + 1e-2 |ref|, relative
L2 <= 1e-2. A row's error is its output's rounding (bf16: 2^-8 of the value at most) and that of its
probabilities (2^-8 of each, so of a mean of values below 5 less than 2e-2). Slots that no
sequence owns hold NaN in bf16 caches.
"""

import ctypes

import numpy as np
import pytest
import torch

from kvcase import Guarded, assert_guards, bits_of, check_attention, guard_cache, slots_for, to_dev_bits
from oracle import fp8, paged, tree
from wavelet_amd import PagedKVCache, _lib, paged_tree_gqa, prefill_gqa, synth

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def random_masks(rng, new, words):
    out = []
    for n in new:
        p = np.array([-1] + [rng.integers(max(0, i - 6), i) for i in range(1, n)])[:n]
        out.append(tree.masks(p, words))
    return np.concatenate(out) if out else np.zeros((0, words), np.int64)


class Case:
    """Cached context written by the oracle, drafted tokens behind it (appended by the call)."""

    def __init__(self, cuda, name, hq, hkv, d, bs, ctx, new, kv="bf16", words=None, seed=0):
        ctx, new = np.asarray(ctx), np.asarray(new)
        lens = ctx + new
        w = self.w = synth.make_decode_workload(name, batch=len(lens), num_kv_heads=hkv, num_q_heads=hq, head_dim=d,
                                                block_size=bs, context_lens=lens)
        self.cuda, self.fp8, self.new, self.lens = cuda, kv == "fp8_e4m3", new, lens
        cs = slots_for(w, np.zeros(w.batch, np.int64), ctx)
        self.slots = slots_for(w, ctx, lens)
        T = int(new.sum())

        def rnd(what, n, h):
            return synth.normal_bf16(synth.stream_key(name, what), (n, h, d))

        self.k, self.v = paged.empty_cache(w.num_blocks, bs, hkv, d, dtype=np.uint8 if self.fp8 else np.uint16,
                                           fill=0 if self.fp8 else 0x7FC0)
        self.ks, self.vs = ((np.zeros((w.num_blocks, hkv), np.float32) for _ in range(2)) if self.fp8 else (None, None))
        self.cache = PagedKVCache(w.num_blocks, bs, hkv, d, kv_dtype=kv, device=cuda)
        self._append(rnd("ck", len(cs), hkv), rnd("cv", len(cs), hkv), cs)
        self.upload()
        self.kn, self.vn, self.q = rnd("nk", T, hkv), rnd("nv", T, hkv), rnd("q", T, hq)
        self.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.words = words or max(1, -(-int(new.max(initial=1)) // 64))
        self.mask = random_masks(np.random.default_rng(seed), new, self.words)

    def _append(self, kb, vb, slots):
        if self.fp8:
            paged.append_fp8(self.k, self.v, self.ks, self.vs, kb, vb, slots)
        else:
            paged.append_bf16(self.k, self.v, kb, vb, slots)

    def upload(self):
        c, dt = self.cache, torch.uint8 if self.fp8 else BF16
        c.k.copy_(to_dev_bits(self.k, dt, self.cuda))
        c.v.copy_(to_dev_bits(self.v, dt, self.cuda))
        if self.fp8:
            c.k_scale.copy_(torch.from_numpy(self.ks))
            c.v_scale.copy_(torch.from_numpy(self.vs))

    def dev(self, x):
        return torch.from_numpy(np.ascontiguousarray(x)).to(self.cuda)

    def args(self):
        return (to_dev_bits(self.q, BF16, self.cuda), self.cache, self.dev(self.w.block_tables),
                self.dev(self.lens.astype(np.int32)), self.dev(self.cu), self.dev(self.mask), self.w.scale)

    def appended(self):
        return dict(key=to_dev_bits(self.kn, BF16, self.cuda), value=to_dev_bits(self.vn, BF16, self.cuda),
                    slot_mapping=self.dev(self.slots))

    def append_host(self):
        self._append(self.kn, self.vn, self.slots)

    def values(self):
        w = self.w
        if self.fp8:
            kf = fp8.dequantize(paged.k_logical(self.k).reshape(w.num_blocks, w.block_size, w.num_kv_heads, w.head_dim),
                                self.ks[:, None, :, None])
            return kf, fp8.dequantize(paged.v_logical(self.v), self.vs[:, None, :, None])
        kl, vl = paged.logical_kv(self.k, self.v)
        return paged.bf16_to_f32(kl), paged.bf16_to_f32(vl)

    def ref(self, **kw):
        a = dict(block_table=self.w.block_tables, seq_lens=self.lens, cu_seqlens_q=self.cu, tree_mask=self.mask,
                 scale=self.w.scale)
        a.update(kw)
        return tree.tree_gqa(paged.bf16_to_f32(self.q), *self.values(), **a)

    def run(self, what, **kw):
        out = paged_tree_gqa(*self.args(), **self.appended(), **kw)
        self.append_host()
        assert np.array_equal(bits_of(self.cache.k), self.k) and np.array_equal(bits_of(self.cache.v), self.v), what
        sinks = kw.get("sinks")
        check_attention(paged.bf16_to_f32(bits_of(out)), self.ref(sinks=None if sinks is None else sinks.cpu().numpy()), what)
        return out


MIX = ([0, 1, 15, 300, 20, 700, 63, 64, 129], [1, 5, 16, 33, 0, 64, 2, 1, 9])


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("hq,hkv,d,bs", [(32, 8, 128, 16), (14, 2, 64, 16), (28, 4, 128, 48), (4, 4, 128, 64),
                                         (8, 1, 64, 32), (16, 4, 128, 128), (8, 2, 64, 256), (20, 1, 128, 16)])
def test_trees(cuda, kv, hq, hkv, d, bs):
    c = Case(cuda, f"tree{kv}{hq}{hkv}{d}{bs}", hq, hkv, d, bs, *MIX, kv)
    c.run("trees")


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("d", [64, 128])
def test_wide_trees_and_long_contexts(cuda, kv, d):
    """Up to 256 nodes (several row groups), contexts cut into chunks, some of which hold drafted keys alone."""
    c = Case(cuda, f"wide{kv}{d}", 8, 2, d, 16, [2300, 0, 5000, 70], [200, 256, 1, 65], kv)
    a = c.run("wide")
    lib = _lib.load()
    need = lib.wkv_tree_workspace_size(4, int(c.fp8), 2, 8, d, 256, 5001)
    assert need > 0
    # without a workspace a sequence's keys stay in one workgroup; the result is the same to rounding
    q, cache, bt, sl, cu, mask, scale = c.args()
    out = Guarded(tuple(a.shape), BF16, cuda)
    rc = lib.wkv_tree_gqa(ctypes.byref(cache.descriptor()), None, 0, 0, None, 0, 0, None, 0, q.data_ptr(), q.stride(0),
                          q.stride(1), out.t.data_ptr(), a.stride(0), a.stride(1), 8, cu.data_ptr(), sl.data_ptr(),
                          bt.data_ptr(), bt.stride(0), bt.shape[1], 4, 256, 5001, mask.data_ptr(), mask.shape[1], scale,
                          None, 0, None, torch.cuda.current_stream(cuda).cuda_stream)
    assert rc == 0
    check_attention(paged.bf16_to_f32(bits_of(out.t)), c.ref(), "one workgroup")
    assert_guards([out], "one workgroup")
    # a workspace just as large as asked for is not written past
    ws = Guarded((need,), torch.uint8, cuda)
    rc = lib.wkv_tree_gqa(ctypes.byref(cache.descriptor()), None, 0, 0, None, 0, 0, None, 0, q.data_ptr(), q.stride(0),
                          q.stride(1), out.t.data_ptr(), a.stride(0), a.stride(1), 8, cu.data_ptr(), sl.data_ptr(),
                          bt.data_ptr(), bt.stride(0), bt.shape[1], 4, 256, 5001, mask.data_ptr(), mask.shape[1], scale,
                          ws.t.data_ptr(), need, None, torch.cuda.current_stream(cuda).cuda_stream)
    assert rc == 0
    assert_guards([out, ws], "workspace")
    assert torch.equal(out.t, a)


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("batch,longest", [(300, 700), (40, 2000), (3, 9000), (1, 600), (1, 4200)])
def test_lines_of_steps(cuda, kv, batch, longest):
    """The steps of all sequences shared between the workgroups: several sequences to a workgroup, several
    workgroups to a sequence, sequences without tokens and without drafts among them."""
    rng = np.random.default_rng(batch + longest)
    ctx, new = rng.integers(0, longest // 3, batch), rng.integers(0, 12, batch)
    ctx[rng.integers(0, batch)], new[rng.integers(0, batch)] = longest, 64
    new[new.sum() == 0] = 3
    c = Case(cuda, f"line{kv}{batch}{longest}", 8, 4, 128, 16, ctx, new, kv)
    c.run("line")


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("longest", [1000, 14000])
def test_many_row_groups(cuda, kv, longest):
    """More row groups than workgroups run at once, of like lengths (whole, one to a workgroup) and with one far
    longer (cut); sequences without drafts and with two row groups among them."""
    rng = np.random.default_rng(longest)
    ctx, new = rng.integers(800, 1000, 150), rng.integers(0, 6, 150)
    ctx[77], new[[3, 100]] = longest, 65
    c = Case(cuda, f"many{kv}{longest}", 8, 4, 64, 16, ctx, new, kv)
    c.run("many")


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
def test_parts_of_which_a_row_sees_nothing_or_nan(cuda, kv):
    """Workgroups whose whole share of a context lies in blocks outside the cache, and ones where every key is NaN."""
    c = Case(cuda, f"parts{kv}", 4, 2, 128, 16, [3000, 3000, 3000], [20, 20, 20], kv)
    c._append(c.kn, c.vn, c.slots)
    nan = c.w.block_tables[1, 40:180]
    if kv == "bf16":
        c.k[nan] = 0x7FC0
    else:
        c.k[nan] = 0x7F
    c.upload()
    bt = c.w.block_tables.copy()
    bt[0, 3:150] = -1
    bt[2, 60:] = c.w.num_blocks  # the drafted tokens' too
    q, cache, _, sl, cu, mask, scale = c.args()
    out = paged.bf16_to_f32(bits_of(paged_tree_gqa(q, cache, c.dev(bt), sl, cu, mask, scale)))
    ref = c.ref(block_table=bt)
    assert np.isnan(ref[20:40]).all() and np.isnan(out[20:40]).all()
    check_attention(out[:20], ref[:20], "context without blocks")
    check_attention(out[40:], ref[40:], "drafts without blocks")


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
def test_chain_is_the_prefill(cuda, kv):
    c = Case(cuda, f"chain{kv}", 16, 8, 128, 16, [100, 0, 1500], [7, 40, 64], kv)
    c.mask = np.concatenate([tree.masks(np.arange(-1, n - 1), 1) for n in c.new])
    out = c.run("chain")
    q, cache, bt, sl, cu, _, scale = c.args()
    torch.testing.assert_close(out.float(), prefill_gqa(q, cache, bt, sl, cu, scale).float(), atol=2e-2, rtol=1e-2)


@pytest.mark.parametrize("ctx", [[0, 3, 700], [64, 128, 2300]])
def test_any_mask_empty_rows_and_bits_past_the_last_node(cuda, ctx):
    c = Case(cuda, f"any{ctx[0]}", 8, 2, 128, 16, ctx, [65, 3, 130], words=4)
    rng = np.random.default_rng(1)
    c.mask = rng.integers(-2**63, 2**63 - 1, c.mask.shape) & rng.integers(-2**63, 2**63 - 1, c.mask.shape)
    c.mask[[0, 5, 66, 68, 100]] = 0
    out = c.run("any mask")
    if ctx[0] == 0:
        assert (out[0] == 0).all() and (out[5] == 0).all()


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
@pytest.mark.parametrize("where", ["k", "v"])
def test_what_is_not_finite_stays_with_the_rows_that_see_it(cuda, kv, where):
    c = Case(cuda, f"nan{kv}{where}", 8, 2, 64, 16, [0, 50, 1200], [20, 33, 64], kv)
    bad = [3, 19, 20, 40, 60, 100]
    x = c.kn if where == "k" else c.vn
    x[bad[0], 0, 5], x[bad[1], 1, 63], x[bad[2], 0, 0] = 0x7FC0, 0x7FC1, 0x7FC0
    if kv == "bf16":  # (fp8 has no infinity: a value too large is held at 448 of its scale)
        x[bad[3], 1, 17], x[bad[4], 0, 2], x[bad[5], 0, 9] = 0x7F80, 0xFF80, 0x7F80
    out = paged.bf16_to_f32(bits_of(paged_tree_gqa(*c.args(), **c.appended())))
    c.append_host()
    with np.errstate(invalid="ignore", over="ignore"):
        ref = c.ref()
    touched = ~np.isfinite(ref)
    assert touched.any() and not touched.all()
    if where == "k":  # a NaN score takes the whole row
        assert np.isnan(out[np.isnan(ref)]).all()
    else:
        np.testing.assert_array_equal(np.isnan(out), np.isnan(ref))
        np.testing.assert_array_equal(out[np.isinf(ref)], ref[np.isinf(ref)].astype(np.float32))
    check_attention(np.where(touched, 0, out), np.where(touched, 0, ref), "the other rows")


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
def test_blocks_outside_the_cache_are_seen_by_no_row(cuda, kv):
    c = Case(cuda, f"bad{kv}", 8, 2, 128, 16, [300, 40, 0, 900], [17, 3, 16, 64], kv)
    c._append(c.kn, c.vn, c.slots)
    c.upload()
    bt = c.w.block_tables.copy()
    bt[0, 2], bt[0, 19], bt[1, :], bt[2, 0], bt[3, 7:40] = -1, 10**6, -5, c.w.num_blocks, 2**31 - 1
    q, cache, _, sl, cu, mask, scale = c.args()
    out = paged_tree_gqa(q, cache, c.dev(bt), sl, cu, mask, scale)
    ref = c.ref(block_table=bt)
    check_attention(paged.bf16_to_f32(bits_of(out)), ref, "bad blocks")
    assert (out[17:36] == 0).all()  # the second and third sequences see nothing


@pytest.mark.parametrize("kv", ["bf16", "fp8_e4m3"])
def test_sinks(cuda, kv):
    c = Case(cuda, f"sink{kv}", 14, 2, 64, 16, [0, 30, 3000], [5, 33, 40], kv)
    sinks = torch.randn(14, device=cuda) * 2
    sinks[0], sinks[1], sinks[2] = -float("inf"), 9.0, -6.0
    c.run("sinks", sinks=sinks)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(cuda, scale):
    """Masked keys stay masked at any scale; scores far apart move the reference maximum."""
    c = Case(cuda, f"scale{scale}", 8, 4, 128, 16, [0, 200, 1500], [33, 20, 64])
    args = c.args()
    out = paged_tree_gqa(*args[:-1], scale, **c.appended())
    c.append_host()
    check_attention(paged.bf16_to_f32(bits_of(out)), c.ref(scale=scale), "scale")


def test_strided_rows_refused_sequences_and_rows_behind_the_last(cuda):
    """q a slice of a fused projection; out strided; sequences of length 0 with rows give zeros; rows past
    cu_seqlens_q's end and everything between the rows stay as they are."""
    c = Case(cuda, "strided", 8, 2, 128, 16, [40, 100, 0], [20, 33, 8])
    g = guard_cache(c.cache)
    q, cache, bt, sl, cu, mask, scale = c.args()
    T = q.shape[0]
    fused = torch.randn((T + 3, 12 * 128), device=cuda).to(BF16)
    fused[:T, :1024] = q.view(T, 1024)
    buf = torch.full((T + 3, 10, 128), 7.0, dtype=BF16, device=cuda)
    more = lambda x, v=0: torch.cat([x, x.new_full((3, *x.shape[1:]), v)])  # noqa: E731
    new = {k: more(v, -1 if k == "slot_mapping" else 0) for k, v in c.appended().items()}
    out = paged_tree_gqa(fused[:, :1024].unflatten(1, (8, 128)), cache, bt, sl, cu, more(mask), scale, out=buf[:, 1:9], **new)
    c.append_host()
    check_attention(paged.bf16_to_f32(bits_of(out[:T])), c.ref(), "strided")
    assert (buf[T:] == 7).all() and (buf[:, 0] == 7).all() and (buf[:, 9] == 7).all()
    sl[1] = 0
    buf.fill_(7.0)
    paged_tree_gqa(fused[:, :1024].unflatten(1, (8, 128)), cache, bt, sl, cu, more(mask), scale, out=buf[:, 1:9])
    assert (buf[20:53, 1:9] == 0).all() and (buf[:20, 1:9] != 7).any() and (buf[T:] == 7).all()
    assert_guards(g, "cache")


def test_one_sequence_one_node_and_nothing(cuda):
    c = Case(cuda, "one", 4, 4, 64, 16, [0], [1])
    out = c.run("one")
    assert torch.equal(out[:, :, :].view(4, 64), to_dev_bits(c.vn, BF16, cuda).view(4, 64))  # its own value
    q, cache, bt, sl, cu, mask, scale = c.args()
    e = paged_tree_gqa(q[:0], cache, bt, sl, cu * 0, mask[:0], scale)
    assert e.shape == (0, 4, 64)
    e = paged_tree_gqa(q[:0], cache, bt[:0], sl[:0], cu[:1] * 0, mask[:0], scale)
    assert e.shape == (0, 4, 64)


def test_captured_steps(cuda):
    """A captured call (append, cut contexts, merge) replayed with other lengths, masks and queries; eager
    calls of another shape between the replays."""
    c = Case(cuda, "graph", 16, 4, 128, 16, [3000, 900, 30], [16, 16, 16])
    other = Case(cuda, "graph2", 16, 4, 128, 16, [4000], [64])
    q, cache, bt, sl, cu, mask, scale = c.args()
    new = c.appended()
    kw = dict(max_query_len=16, max_seq_len=3100)
    paged_tree_gqa(q, cache, bt, sl, cu, mask, scale, **new, **kw)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_tree_gqa(q, cache, bt, sl, cu, mask, scale, out=out, **new, **kw)
    for i in range(4):
        q.normal_()
        mask.copy_(c.dev(random_masks(np.random.default_rng(i), c.new, 1)))
        sl.copy_(c.dev((c.lens - i).astype(np.int32)))
        new["slot_mapping"].copy_(c.dev(slots_for(c.w, c.lens - i - c.new, c.lens - i)))
        graph.replay()
        other.run("between") if i == 1 else None
        got = out.clone()
        want = paged_tree_gqa(q, cache, bt, sl, cu, mask, scale, **new, **kw)
        torch.cuda.synchronize()
        assert torch.equal(got, want), f"replay {i}"


def test_on_another_stream(cuda):
    c = Case(cuda, "stream", 8, 2, 128, 16, [2500, 10], [30, 5])
    args, new = c.args(), c.appended()
    s = torch.cuda.Stream(cuda)
    s.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(s):
        out = paged_tree_gqa(*args, **new)
    torch.cuda.current_stream(cuda).wait_stream(s)
    c.append_host()
    check_attention(paged.bf16_to_f32(bits_of(out)), c.ref(), "stream")


def test_two_calls_at_once(cuda):
    """Calls on two streams that share nothing but the queries give what each gives alone."""
    a = Case(cuda, "both0", 8, 2, 128, 16, [6000, 900], [64, 40])
    b = Case(cuda, "both1", 8, 2, 128, 16, [5000], [50])
    alone = [paged_tree_gqa(*c.args(), **c.appended()) for c in (a, b)]
    calls = [(c.args(), c.appended()) for c in (a, b)]
    streams = [torch.cuda.Stream(cuda) for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (args, new) in enumerate(calls):
            with torch.cuda.stream(streams[i]):
                got[i].append(paged_tree_gqa(*args, max_query_len=64, max_seq_len=6100, **new))
    torch.cuda.synchronize()
    for want, outs in zip(alone, got):
        for out in outs:
            torch.testing.assert_close(out.float(), want.float(), atol=2e-2, rtol=1e-2)
            assert torch.equal(out, outs[0])


def test_refusals(cuda):
    c = Case(cuda, "refuse", 8, 2, 128, 16, [10], [4])
    names = ("q", "cache", "block_table", "seq_lens", "cu_seqlens_q", "tree_mask", "scale")
    ok = dict(zip(names, c.args()))
    new = c.appended()
    q, mask = ok["q"], ok["tree_mask"]
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(q=q[:, :, :64]), dict(q=q[:, :7]), dict(cache=None),
                dict(seq_lens=ok["seq_lens"].long()), dict(cu_seqlens_q=ok["cu_seqlens_q"][:1]),
                dict(cu_seqlens_q=ok["cu_seqlens_q"].long()), dict(tree_mask=mask.int()), dict(tree_mask=mask[:2]),
                dict(tree_mask=mask[:, 0]), dict(tree_mask=mask.expand(4, 5)), dict(scale=float("inf")),
                dict(key=new["key"]), dict(key=new["key"][:2], value=new["value"], slot_mapping=new["slot_mapping"]),
                dict(out=torch.empty_like(q).float()), dict(out=torch.empty_like(q)[:2]),
                dict(out=torch.empty_like(q, device="cpu")), dict(sinks=torch.zeros(7, device=cuda))):
        with pytest.raises(ValueError):
            paged_tree_gqa(**{**ok, **bad})
    before = c.cache.k.clone()
    with pytest.raises(ValueError):  # refused: nothing is appended
        paged_tree_gqa(**{**ok, "scale": float("nan")}, **new)
    assert torch.equal(c.cache.k.view(torch.int16), before.view(torch.int16))
