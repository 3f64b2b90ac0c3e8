// Keys and values into the paged cache with the norm of heads and the rotary
// positions on the way, and the queries to the attention, in one launch (gfx950).
// The mathematics of heads: norm_rotary_dev.h; the fp8 rule: kv_append_dev.h.
//
// The workgroups of a launch have one of two roles. Rows: a tile of tokens, its angles in
// LDS, and the heads that are stored as rows: queries, the keys of a bf16 cache, whose
// 16-byte runs are the cache's own pieces, and the shared key of a latent
// cache. The rest: values (bf16: a window of 64 tokens of one head, transposed through LDS; few
// tokens: an element at a time), keys and values (fp8, run by run, because a block's scale follows from all of
// its new keys: a wave norms and turns 16 of them into LDS and codes them from there),
// or a latent cache's compressed entries, normed.
#include <type_traits>

#include "kv_append_dev.h"
#include "norm_rotary_dev.h"

namespace wkv {

constexpr int kThreads = 256, kWaves = kThreads / 64;

struct AppendArgs {
  HeadRows q;  // y: the queries' result
  const uint16_t *key, *val;
  int64_t kst, ksh, vst, vsh;
  const int64_t *slots;
  HeadNorm n;
  Angles a;
  RowUnits r;
  int64_t tokens;
  int Hq, Hk;
  void *kc, *vc;
  float *ks, *vs;
  int BS;
  int64_t NB;
  int rows;           // heads of the rows role: queries, and a bf16 cache's keys
  int tile;           // its tokens of a workgroup
  FastDiv per, last;  // its heads of a workgroup; of a token's last one
  FastDiv splits;     // its workgroups of a tile
  int64_t row_wgs;    // all of them
  int window;         // tokens of a workgroup of the other role
};

__device__ __forceinline__ bool block_of(int64_t slot, int BS, int64_t NB, int64_t &blk, int &off) {
  blk = slot / BS;
  off = static_cast<int>(slot - blk * BS);
  return slot >= 0 && blk < NB;
}

template <int V, bool INTER, bool PAGED_K>
__device__ __forceinline__ void rows_role(const AppendArgs &a, int64_t wg, float2 *turn) {
  typedef typename VecOf<__bf16, V>::type Vec;
  const int64_t tile = wg / a.splits.d;
  const int split = static_cast<int>(wg - tile * a.splits.d);
  const int64_t t0 = tile * a.tile;
  const int nt = a.tokens - t0 < a.tile ? static_cast<int>(a.tokens - t0) : a.tile;
  tile_angles(a.a, t0, nt, kThreads, turn);
  __syncthreads();
  norm_turn_rows<__bf16, V, INTER, 1, 2, false>(
      a.r, a.n, a.Hq, turn, nt, split + 1 == a.splits.d ? a.last : a.per, split * a.per.d, kThreads,
      [&](int t, int h) {
        if (PAGED_K && h >= a.Hq) {
          int64_t blk;
          int off;
          if (!block_of(a.slots[t0 + t], a.BS, a.NB, blk, off)) return static_cast<const __bf16 *>(nullptr);
          return reinterpret_cast<const __bf16 *>(a.key) + (t0 + t) * a.kst + (h - a.Hq) * a.ksh;
        }
        return static_cast<const __bf16 *>(a.q.x) + (t0 + t) * a.q.xt + h * a.q.xh;
      },
      [&](int t, int h, int e, Vec v) {
        __bf16 *y;
        if (PAGED_K && h >= a.Hq) {
          int64_t blk;
          int off;
          block_of(a.slots[t0 + t], a.BS, a.NB, blk, off);
          y = static_cast<__bf16 *>(a.kc) + (((blk * a.Hk + h - a.Hq) * (a.r.D / 8) + (e >> 3)) * a.BS + off) * 8 + (e & 7);
        } else {
          y = static_cast<__bf16 *>(a.q.y) + (t0 + t) * a.q.yt + h * a.q.yh + e;
        }
        *reinterpret_cast<Vec *>(y) = v;
      });
}

// ---------------------------------------------------------------------------
// bf16 values.
constexpr int kValueWindow = 64;
constexpr int64_t kValueWindowTokens = 256;  // below this the values go element by element, over more workgroups

template <int D>
__device__ __forceinline__ void values_role(const AppendArgs &a, int64_t wg, uint8_t *lds) {
  constexpr int C = D / 8;
  uint16_t *vc = static_cast<uint16_t *>(a.vc);
  if (a.window == 1) {  // an item a thread: 8 elements of a token's head
    const int64_t i = wg * kThreads + threadIdx.x;
    if (i >= a.tokens * a.Hk * C) return;
    const int c = static_cast<int>(i % C);
    const int64_t th = i / C;
    const int h = static_cast<int>(th % a.Hk);
    const int64_t t = th / a.Hk;
    int64_t blk;
    int off;
    if (!block_of(a.slots[t], a.BS, a.NB, blk, off)) return;
    const u32x4 v = *reinterpret_cast<const u32x4 *>(a.val + t * a.vst + h * a.vsh + c * 8);
    uint16_t *y = vc + ((blk * a.Hk + h) * D + c * 8) * a.BS + off;
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j * a.BS] = static_cast<uint16_t>(v[j >> 1] >> (16 * (j & 1)));
    return;
  }
  // A window's values through LDS; tokens in groups of 8: one whose slots are consecutive and
  // start 8-aligned in a block is stored 16 bytes of a d row at a time, another token by token.
  constexpr int RP = D * 2 + 8;  // pitch of a token's row in LDS
  constexpr int NG = kValueWindow / 8;
  int64_t *gslot = reinterpret_cast<int64_t *>(lds + kValueWindow * RP);
  const int64_t w = wg / a.Hk, t0 = w * kValueWindow;
  const int h = static_cast<int>(wg - w * a.Hk), tid = threadIdx.x;
#pragma unroll
  for (int k = 0; k < kValueWindow * C / kThreads; ++k) {
    const int t = tid / C + k * (kThreads / C), c = tid % C;
    if (t0 + t < a.tokens) {
      const u32x4 v = *reinterpret_cast<const u32x4 *>(a.val + (t0 + t) * a.vst + h * a.vsh + c * 8);
      uint32_t *l = reinterpret_cast<uint32_t *>(lds + t * RP + c * 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) l[j] = v[j];
    }
  }
  if (tid < NG) {
    const int64_t ta = t0 + 8 * tid;
    int64_t first = -1;
    if (ta + 7 < a.tokens) {
      int64_t s[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = a.slots[ta + j];
      bool run = s[0] >= 0 && s[0] / a.BS < a.NB && (s[0] % a.BS) % 8 == 0;
#pragma unroll
      for (int j = 1; j < 8; ++j) run = run && s[j] == s[0] + j;
      if (run) first = s[0];
    }
    gslot[tid] = first;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < NG * D / kThreads; ++k) {
    const int i = tid + kThreads * k;
    const int g = 2 * (i / (2 * D)) + (i & 1), d = (i >> 1) % D;
    const int64_t first = gslot[g];
    if (first >= 0) {
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = *reinterpret_cast<const uint16_t *>(lds + (8 * g + 2 * j) * RP + 2 * d);
        const uint32_t hi = *reinterpret_cast<const uint16_t *>(lds + (8 * g + 2 * j + 1) * RP + 2 * d);
        o[j] = lo | (hi << 16);
      }
      const int64_t blk = first / a.BS;
      *reinterpret_cast<u32x4 *>(vc + ((blk * a.Hk + h) * D + d) * a.BS + (first - blk * a.BS)) = u32x4{o[0], o[1], o[2], o[3]};
    } else {
      for (int j = 0; j < 8; ++j) {
        const int t = 8 * g + j;
        if (t0 + t >= a.tokens) break;
        int64_t blk;
        int off;
        if (!block_of(a.slots[t0 + t], a.BS, a.NB, blk, off)) continue;
        vc[((blk * a.Hk + h) * D + d) * a.BS + off] = *reinterpret_cast<const uint16_t *>(lds + t * RP + 2 * d);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// fp8 keys and values.
constexpr int kPiece = 16;  // tokens of a run taken at a time

template <int D>
constexpr int kKeyPitch = D + 8;  // of a key in LDS, in elements

// Piece p0 of a run (tokens t + p0 ..): its n keys of head h normed and turned into the wave's rows of LDS.
template <int D, int V, bool INTER>
__device__ __forceinline__ void stage_keys(const AppendArgs &a, const float2 *turn, int64_t t, int n, int h,
                                           uint16_t *rows) {
  typedef typename VecOf<__bf16, V>::type Vec;
  const int lane = threadIdx.x & 63, lanes = 1 << a.r.log_lanes, group = lane >> a.r.log_lanes, u = lane & (lanes - 1);
  const int groups = 64 >> a.r.log_lanes;
  int e0 = 0, e1 = 0;
  if (u < a.r.units) unit_runs<V, INTER>(a.r, u, e0, e1);
  float w0[V], w1[V];
  load_weights<__bf16, V>(a.n, a.n.kw, h * a.n.kws + e0, w0);
  load_weights<__bf16, V>(a.n, a.n.kw, h * a.n.kws + e1, w1);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the rows of the piece before have been read
  __builtin_amdgcn_wave_barrier();
  for (int i0 = 0; i0 < n; i0 += groups) {  // uniform
    const int i = i0 + group;
    const bool in = i < n && u < a.r.units;
    float f0[V], f1[V], ss = 0.f;
    Vec x0 = Vec{}, x1 = Vec{};
    if (in) {
      const __bf16 *x = reinterpret_cast<const __bf16 *>(a.key) + (t + i) * a.kst + h * a.ksh;
      x0 = *reinterpret_cast<const Vec *>(x + e0);
      x1 = *reinterpret_cast<const Vec *>(x + e1);
    }
    widen<V, __bf16>(x0, f0);
    widen<V, __bf16>(x1, f1);
#pragma unroll
    for (int v = 0; v < V; ++v) ss = __builtin_fmaf(f0[v], f0[v], __builtin_fmaf(f1[v], f1[v], ss));
    ss = group_sum(ss, a.r.log_lanes);
    if (!in) continue;
    const float inv = a.n.on ? rsqrtf(__builtin_fmaf(ss, 1.f / static_cast<float>(D), a.n.eps)) : 1.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      f0[v] *= inv * w0[v];
      f1[v] *= inv * w1[v];
    }
    turn_unit<V, INTER>(turn + i * a.r.half, a.r.half, e0, e1, f0, f1);
    Vec o0, o1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      o0[v] = static_cast<__bf16>(f0[v]);
      o1[v] = static_cast<__bf16>(f1[v]);
    }
    *reinterpret_cast<Vec *>(rows + i * kKeyPitch<D> + e0) = o0;
    *reinterpret_cast<Vec *>(rows + i * kKeyPitch<D> + e1) = o1;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A run of r tokens from t on (block blk, the first at offset `first`): the wave's head h, as
// fp8_append_run_kv appends it, its keys from LDS. Every wave of the workgroup calls it (the
// pieces' angles are the workgroup's); active: the wave has a head.
template <int D, int V, bool INTER>
__device__ __forceinline__ void append_run(const AppendArgs &a, float2 *turn, uint16_t *rows, int64_t t, int r,
                                           int64_t blk, int first, int h, bool active) {
  constexpr int NC = D / 64, RV = D / 64;
  uint8_t *kc = static_cast<uint8_t *>(a.kc), *vc = static_cast<uint8_t *>(a.vc);
  const int lane = threadIdx.x & 63, m = lane & 15, H = a.Hk, BS = a.BS;
  const int64_t si = blk * H + h;
  float sk_old = 0.f, sv_old = 0.f;
  if (active && first != 0) {
    sk_old = a.ks[si];
    sv_old = a.vs[si];
  }
  u32x4 kw[NC][2];
  uint32_t vw[kPiece];
  int off = 0;  // offset in the block of the piece's token m
  auto load = [&](int p0) __attribute__((always_inline)) {
    const int n = r - p0 < kPiece ? r - p0 : kPiece, last = n - 1;
    __syncthreads();  // the angles before have been read
    tile_angles(a.a, t + p0, n, kThreads, turn);
    __syncthreads();
    if (!active) return;
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
      const uint16_t *p = a.val + (t + p0 + (i < last ? i : last)) * a.vst + h * a.vsh + RV * lane;
      if constexpr (RV == 2)
        vw[i] = *reinterpret_cast<const uint32_t *>(p);
      else
        vw[i] = *p;
    }
    const int mm = m < last ? m : last;
    off = static_cast<int>(a.slots[t + p0 + mm] - blk * BS);
    stage_keys<D, V, INTER>(a, turn, t + p0, n, h, rows);
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const uint16_t *p = rows + mm * kKeyPitch<D> + 16 * ((lane >> 4) + 4 * j);
      kw[j][0] = *reinterpret_cast<const u32x4 *>(p);
      kw[j][1] = *reinterpret_cast<const u32x4 *>(p + 8);
    }
  };
  uint32_t ka = 0u, va = 0u;  // largest magnitude bits, as bf16; a NaN counts as none, and is remembered
  bool nan = false;
  auto mag = [&](uint32_t x, uint32_t w) __attribute__((always_inline)) {
    const uint32_t lo = w & 0x7fffu, hi = (w >> 16) & 0x7fffu;
    nan = nan || lo > 0x7f80u || hi > 0x7f80u;
    return max(x, max(lo > 0x7f80u ? 0u : lo, hi > 0x7f80u ? 0u : hi));
  };
  for (int p0 = 0; p0 < r; p0 += kPiece) {  // uniform
    load(p0);
    if (!active) continue;
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) ka = mag(ka, kw[j][q][e]);
#pragma unroll
    for (int i = 0; i < kPiece; ++i) va = mag(va, vw[i]);
  }
  ka = wave_reduce(ka, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
  va = wave_reduce(va, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
  const bool any_nan = __any(nan);
  float sk = pow2_scale(__uint_as_float(ka << 16)), sv = pow2_scale(__uint_as_float(va << 16));
  if (active && first != 0) {
    if (sk > sk_old)
      fp8_reencode_block<D, false>(kc, blk, h, H, BS, first, sk_old / sk);
    else
      sk = sk_old;
    if (sv > sv_old)
      fp8_reencode_block<D, true>(vc, blk, h, H, BS, first, sv_old / sv);
    else
      sv = sv_old;
  }
  const float ik = 1.0f / sk, iv = 1.0f / sv;  // exact: powers of two
  auto q = [](uint32_t bits, float inv) {
    float v = __uint_as_float(bits << 16) * inv;
    v = (v != v) ? v : fminf(fmaxf(v, -448.0f), 448.0f);
    return e4m3_encode(v);
  };
  auto pack8 = [&](uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, float inv) __attribute__((always_inline)) {
    if (!any_nan) return e4m3_pack8(w0, w1, w2, w3, inv);  // uniform
    u32x2 o;
    o[0] = q(w0 & 0xffffu, inv) | (q(w0 >> 16, inv) << 8) | (q(w1 & 0xffffu, inv) << 16) | (q(w1 >> 16, inv) << 24);
    o[1] = q(w2 & 0xffffu, inv) | (q(w2 >> 16, inv) << 8) | (q(w3 & 0xffffu, inv) << 16) | (q(w3 >> 16, inv) << 24);
    return o;
  };
  for (int p0 = 0; p0 < r; p0 += kPiece) {
    if (r > kPiece) load(p0);
    if (!active) continue;
    const int n = r - p0 < kPiece ? r - p0 : kPiece;
    if (m < n) {
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const u32x2 x = pack8(kw[j][0][0], kw[j][0][1], kw[j][0][2], kw[j][0][3], ik);
        const u32x2 y = pack8(kw[j][1][0], kw[j][1][1], kw[j][1][2], kw[j][1][3], ik);
        *reinterpret_cast<u32x4 *>(kc + fp8_k_index<D>(blk, h, H, BS, off, 16 * ((lane >> 4) + 4 * j))) =
            u32x4{x[0], x[1], y[0], y[1]};
      }
    }
    // consecutive offsets from a 16-aligned one on: a d row's 16 tokens in one store
    const int off0 = __builtin_amdgcn_readfirstlane(off);
    const bool whole = n == kPiece && off0 % kPiece == 0 && __all(off == off0 + m);
#pragma unroll
    for (int rr = 0; rr < RV; ++rr) {
      uint8_t *row = vc + fp8_v_index<D>(blk, h, H, BS, 0, RV * lane + rr);
      auto pair = [&](int i) { return ((vw[i] >> (16 * rr)) & 0xffffu) | (((vw[i + 1] >> (16 * rr)) & 0xffffu) << 16); };
      const u32x2 c0 = pack8(pair(0), pair(2), pair(4), pair(6), iv);
      const u32x2 c1 = pack8(pair(8), pair(10), pair(12), pair(14), iv);
      if (whole) {
        *reinterpret_cast<u32x4 *>(row + off0) = u32x4{c0[0], c0[1], c1[0], c1[1]};
      } else {
#pragma unroll
        for (int i = 0; i < kPiece; ++i)
          if (i < n) row[__builtin_amdgcn_readlane(off, i)] = static_cast<uint8_t>((i < 8 ? c0 : c1)[(i & 7) >> 2] >> (8 * (i & 3)));
      }
    }
  }
  if (active && lane == 0) {
    a.ks[si] = sk;
    a.vs[si] = sv;
  }
}

// A window's runs, four heads a workgroup, one a wave.
template <int D, int V, bool INTER>
__device__ __forceinline__ void fp8_role(const AppendArgs &a, int64_t wg, float2 *turn, uint16_t *all_rows) {
  const int chunks = (a.Hk + kWaves - 1) / kWaves;
  const int64_t w = wg / chunks, t0 = w * a.window;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int h = static_cast<int>(wg - w * chunks) * kWaves + wave;
  const bool active = h < a.Hk;
  uint16_t *rows = all_rows + wave * kPiece * kKeyPitch<D>;
  // lane l: token t0 - 1 + l, its block (-1: none); the window and, behind it, up to 63 - window tokens
  auto block_at = [&](int64_t tok) {
    int64_t blk;
    int off;
    return tok >= 0 && tok < a.tokens && block_of(a.slots[tok], a.BS, a.NB, blk, off) ? static_cast<int>(blk) : -1;
  };
  const int mine = block_at(t0 - 1 + lane);
  const int before = __shfl_up(mine, 1, 64);
  const uint64_t cont = __ballot(lane > 0 && mine >= 0 && mine == before);
  uint64_t starts = __ballot(lane > 0 && lane <= a.window && mine >= 0 && mine != before);
  while (starts != 0) {  // uniform, and the same in every wave
    const int i = __builtin_ctzll(starts);
    starts &= starts - 1;
    const int blk = __builtin_amdgcn_readlane(mine, i);
    const uint64_t after = i < 63 ? ~(cont >> (i + 1)) : 1ull;  // (the bits shifted in end the run)
    int r = 1 + __builtin_ctzll(after);
    if (i + r == 64) {  // the view's end: the tokens behind it
      for (;;) {
        const uint64_t same = __ballot(block_at(t0 - 1 + i + r + lane) == blk);
        const int more = ~same == 0 ? 64 : __builtin_ctzll(~same);
        r += more;
        if (more < 64) break;
      }
    }
    const int64_t t = t0 - 1 + i;
    const int first = static_cast<int>(a.slots[t] - static_cast<int64_t>(blk) * a.BS);
    append_run<D, V, INTER>(a, turn, rows, t, r, blk, first, h, active);
  }
}

template <int D, int V, bool INTER, bool FP8>
__global__ __launch_bounds__(kThreads) void rotary_append_kernel(AppendArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int64_t wg = blockIdx.x;
  if (wg < a.row_wgs)
    rows_role<V, INTER, !FP8>(a, wg, reinterpret_cast<float2 *>(lds));
  else if (FP8)
    fp8_role<D, V, INTER>(a, wg - a.row_wgs, reinterpret_cast<float2 *>(lds + kWaves * kPiece * kKeyPitch<D> * 2),
                          reinterpret_cast<uint16_t *>(lds));
  else
    values_role<D>(a, wg - a.row_wgs, lds);
}

// ---------------------------------------------------------------------------
// The latent cache: rows of rope_dim (every query head's, and the shared key as one more), and the compressed
// entries, a wave each.
struct LatentArgs {
  HeadRows q;
  const __bf16 *kvc, *kpe;
  int64_t kvc_st, kpe_st;
  const int64_t *slots;
  HeadNorm n;  // of the entries: kw
  Angles a;
  RowUnits r;
  int64_t tokens;
  int heads, rank;
  __bf16 *latent;
  int BS;
  int64_t NB;
  int tile;
  FastDiv per, last, splits;
  int64_t row_wgs;
};

template <int V, bool INTER>
__global__ __launch_bounds__(kThreads) void mla_rotary_append_kernel(LatentArgs a) {
  typedef typename VecOf<__bf16, V>::type Vec;
  extern __shared__ float2 turn[];
  const int width = a.rank + a.r.D;
  const int64_t wg = blockIdx.x;
  if (wg < a.row_wgs) {
    const int64_t tile = wg / a.splits.d, t0 = tile * a.tile;
    const int split = static_cast<int>(wg - tile * a.splits.d);
    const int nt = a.tokens - t0 < a.tile ? static_cast<int>(a.tokens - t0) : a.tile;
    tile_angles(a.a, t0, nt, kThreads, turn);
    __syncthreads();
    const HeadNorm none{};
    norm_turn_rows<__bf16, V, INTER, 1, 2, false>(
        a.r, none, a.heads, turn, nt, split + 1 == a.splits.d ? a.last : a.per, split * a.per.d, kThreads,
        [&](int t, int h) {
          if (h < a.heads) return static_cast<const __bf16 *>(a.q.x) + (t0 + t) * a.q.xt + h * a.q.xh;
          int64_t blk;
          int off;
          if (!block_of(a.slots[t0 + t], a.BS, a.NB, blk, off)) return static_cast<const __bf16 *>(nullptr);
          return a.kpe + (t0 + t) * a.kpe_st;
        },
        [&](int t, int h, int e, Vec v) {
          __bf16 *y = h < a.heads ? static_cast<__bf16 *>(a.q.y) + (t0 + t) * a.q.yt + h * a.q.yh + e
                                  : a.latent + a.slots[t0 + t] * width + a.rank + e;
          *reinterpret_cast<Vec *>(y) = v;
        });
    return;
  }
  const int lane = threadIdx.x & 63;
  const int64_t t = (wg - a.row_wgs) * kWaves + (threadIdx.x >> 6);
  if (t >= a.tokens) return;  // a whole wave; nothing below waits for another
  int64_t blk;
  int off;
  if (!block_of(a.slots[t], a.BS, a.NB, blk, off)) return;
  typedef typename VecOf<__bf16, 8>::type Vec8;
  const __bf16 *x = a.kvc + t * a.kvc_st;
  __bf16 *y = a.latent + a.slots[t] * width;
  float f[8], ss = 0.f, inv = 1.f;
  if (a.n.on) {
    for (int e = 8 * lane; e < a.rank; e += 512) {
      widen<8, __bf16>(*reinterpret_cast<const Vec8 *>(x + e), f);
#pragma unroll
      for (int v = 0; v < 8; ++v) ss = __builtin_fmaf(f[v], f[v], ss);
    }
    inv = rsqrtf(__builtin_fmaf(wave_sum(ss), 1.f / static_cast<float>(a.rank), a.n.eps));
  }
  for (int e = 8 * lane; e < a.rank; e += 512) {
    float w[8];
    Vec8 o;
    widen<8, __bf16>(*reinterpret_cast<const Vec8 *>(x + e), f);
    load_weights<__bf16, 8>(a.n, a.n.kw, e, w);
#pragma unroll
    for (int v = 0; v < 8; ++v) o[v] = static_cast<__bf16>(f[v] * (inv * w[v]));
    *reinterpret_cast<Vec8 *>(y + e) = o;
  }
}

}  // namespace wkv

using namespace wkv;

namespace {

int check_rows16(const void *p, int64_t st, int64_t sh, const char *name) {
  WKV_CHECK_ARG(p != nullptr && aligned16(p), "%s must be non-NULL and 16-byte aligned", name);
  WKV_CHECK_ARG(st >= 0 && sh >= 0 && st % 8 == 0 && sh % 8 == 0, "%s strides must be non-negative multiples of 8 (got %lld, %lld)",
                name, (long long)st, (long long)sh);
  return WKV_OK;
}

// The rows role's grid: tiles of tokens, and with too few of them for the chip, their heads over more workgroups.
struct RowGrid {
  int tile, per, splits, last;
  int64_t wgs;
  RowGrid(int64_t tokens, int heads, int half, int log_lanes) {
    tile = half > 0 && 1024 / half < 16 ? 1024 / half : 16;
    while (tile > 1 && (tokens + tile - 1) / tile < 1024) tile /= 2;
    const int64_t tiles = (tokens + tile - 1) / tile;
    const int groups = kThreads >> log_lanes;
    const int64_t want = (1024 + tiles - 1) / tiles, most = (heads + groups - 1) / groups;
    int n = static_cast<int>(want < most ? want : most);
    if (n < 1) n = 1;
    per = (heads + n - 1) / n;
    if (per < 1) per = 1;
    splits = heads > 0 ? (heads + per - 1) / per : 1;
    last = heads - (splits - 1) * per;
    wgs = heads > 0 ? tiles * splits : 0;
  }
};

}  // namespace

extern "C" int wkv_rotary_append(const wkv_cache_t *cache, const void *key, int64_t key_stride_t, int64_t key_stride_h,
                                 const void *value, int64_t value_stride_t, int64_t value_stride_h,
                                 const int64_t *slot_mapping, const void *q, int64_t q_stride_t, int64_t q_stride_h,
                                 void *q_out, int64_t qo_stride_t, int64_t qo_stride_h, int32_t num_q_heads,
                                 const wkv_head_norm_t *norm, const wkv_rotary_t *rotary, int64_t num_tokens,
                                 void *stream) {
  if (const int rc = check_cache(cache, -1)) return rc;
  WKV_CHECK_ARG(num_tokens >= 0 && num_tokens <= INT32_MAX, "num_tokens must be in [0, 2^31) (got %lld)",
                (long long)num_tokens);
  const int D = cache->head_dim, Hk = cache->num_kv_heads;
  WKV_CHECK_ARG(num_q_heads >= 0 && num_q_heads <= 65535 && Hk <= 65535, "head counts must be in [0, 65535]");
  WKV_CHECK_ARG(cache->num_blocks <= INT32_MAX, "num_blocks must be below 2^31 (got %lld)", (long long)cache->num_blocks);
  WKV_CHECK_ARG(norm != nullptr || rotary != nullptr, "a norm or a rotation must be given (wkv_append has neither)");
  if (norm != nullptr)
    if (const int rc = check_head_norm(norm, 1)) return rc;
  if (rotary != nullptr)
    if (const int rc = check_rotary(rotary, D, num_tokens)) return rc;
  if (num_tokens == 0) return WKV_OK;
  WKV_CHECK_ARG(slot_mapping != nullptr && reinterpret_cast<uintptr_t>(slot_mapping) % 8 == 0, "slot_mapping must be int64");
  if (const int rc = check_rows16(key, key_stride_t, key_stride_h, "key")) return rc;
  if (const int rc = check_rows16(value, value_stride_t, value_stride_h, "value")) return rc;
  WKV_CHECK_ARG(num_q_heads == 0 || (q != nullptr && q_out != nullptr && reinterpret_cast<uintptr_t>(q) % 2 == 0 &&
                    reinterpret_cast<uintptr_t>(q_out) % 2 == 0 && q_stride_t >= 0 && q_stride_h >= 0 &&
                    qo_stride_t >= 0 && qo_stride_h >= 0),
                "q and its output must be non-NULL, aligned to their elements, their strides non-negative");
  const bool fp8 = cache->kv_dtype == WKV_KV_FP8_E4M3;
  const int half = rotary != nullptr ? rotary->rotary_dim / 2 : 0;
  const bool inter = rotary != nullptr && rotary->interleaved != 0;
  Widths w(2, D, half, inter);
  if (num_q_heads > 0) {
    w.rows(q, q_stride_t, q_stride_h);
    w.rows(q_out, qo_stride_t, qo_stride_h);
  }
  if (norm != nullptr) {
    const int wsz = norm->weight_dtype == 0 ? 4 : 2;
    if (num_q_heads > 0) w.weights(norm->q_weight, norm->q_weight_stride_h, wsz);
    w.weights(norm->k_weight, norm->k_weight_stride_h, wsz);
  }
  if (w.v < 8) w.v = 1;
  AppendArgs a{};
  a.q = HeadRows{q, q_out, q_stride_t, q_stride_h, qo_stride_t, qo_stride_h};
  a.key = static_cast<const uint16_t *>(key);
  a.val = static_cast<const uint16_t *>(value);
  a.kst = key_stride_t;
  a.ksh = key_stride_h;
  a.vst = value_stride_t;
  a.vsh = value_stride_h;
  a.slots = slot_mapping;
  a.n = head_norm(norm);
  a.a = angles(rotary);
  a.r = row_units(D, half, w.v);
  a.tokens = num_tokens;
  a.Hq = num_q_heads;
  a.Hk = Hk;
  a.kc = cache->k;
  a.vc = cache->v;
  a.ks = cache->k_scale;
  a.vs = cache->v_scale;
  a.BS = cache->block_size;
  a.NB = cache->num_blocks;
  a.rows = num_q_heads + (fp8 ? 0 : Hk);
  const RowGrid g(num_tokens, a.rows, half, a.r.log_lanes);
  a.tile = g.tile;
  a.per = fast_div(g.per);
  a.last = fast_div(g.last > 0 ? g.last : 1);
  a.splits = fast_div(g.splits);
  a.row_wgs = g.wgs;
  size_t lds = static_cast<size_t>(g.tile) * half * sizeof(float2);
  int64_t rest;
  if (fp8) {
    // a window of 16 tokens for prompts, of one where there is a token a sequence
    a.window = num_tokens >= 4096 ? 16 : num_tokens >= 1024 ? 4 : 1;
    rest = (num_tokens + a.window - 1) / a.window * ((Hk + kWaves - 1) / kWaves);
    const size_t need = kWaves * kPiece * (D + 8) * 2 + static_cast<size_t>(kPiece) * half * sizeof(float2);
    lds = lds > need ? lds : need;
  } else if (num_tokens < kValueWindowTokens) {
    a.window = 1;
    rest = (num_tokens * Hk * (D / 8) + kThreads - 1) / kThreads;
  } else {
    a.window = kValueWindow;
    rest = (num_tokens + kValueWindow - 1) / kValueWindow * Hk;
    const size_t need = kValueWindow * (D * 2 + 8) + kValueWindow / 8 * sizeof(int64_t);
    lds = lds > need ? lds : need;
  }
  WKV_CHECK_ARG(a.row_wgs + rest <= INT32_MAX, "too many tokens and heads for one launch");
  const unsigned grid = static_cast<unsigned>(a.row_wgs + rest);
  auto s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto d, auto v, auto in) {
    constexpr int DD = decltype(d)::value, VV = decltype(v)::value;
    constexpr bool IN = decltype(in)::value;
    if (fp8) rotary_append_kernel<DD, VV, IN, true><<<grid, kThreads, lds, s>>>(a);
    else rotary_append_kernel<DD, VV, IN, false><<<grid, kThreads, lds, s>>>(a);
  };
  auto layout = [&](auto d, auto v) {
    if (inter) launch(d, v, std::true_type{}); else launch(d, v, std::false_type{});
  };
  auto width = [&](auto d) {
    if (w.v == 8) layout(d, std::integral_constant<int, 8>{}); else layout(d, std::integral_constant<int, 1>{});
  };
  if (D == 128) width(std::integral_constant<int, 128>{}); else width(std::integral_constant<int, 64>{});
  WKV_CHECK_LAUNCH("rotary_append");
  return WKV_OK;
}

extern "C" int wkv_mla_rotary_append(const wkv_mla_cache_t *cache, const void *kv_c, int64_t kv_c_stride,
                                     const void *k_pe, int64_t k_pe_stride, const int64_t *slot_mapping,
                                     const void *q_pe, int64_t q_stride_t, int64_t q_stride_h, void *q_out,
                                     int64_t qo_stride_t, int64_t qo_stride_h, int32_t num_heads,
                                     const wkv_head_norm_t *kv_norm, const wkv_rotary_t *rotary, int64_t num_tokens,
                                     void *stream) {
  if (const int rc = check_mla_cache(cache)) return rc;
  WKV_CHECK_ARG(num_tokens >= 0 && num_tokens <= INT32_MAX, "num_tokens must be in [0, 2^31) (got %lld)",
                (long long)num_tokens);
  WKV_CHECK_ARG(num_heads >= 0 && num_heads <= 65535, "num_heads must be in [0, 65535]");
  const int D = cache->rope_dim;
  WKV_CHECK_ARG(D > 0 && D <= WKV_ROTARY_MAX_DIM, "rope_dim must be in [8, %d] (got %d)", WKV_ROTARY_MAX_DIM, D);
  WKV_CHECK_ARG(rotary != nullptr, "rotary must be given (wkv_mla_append has none)");
  if (const int rc = check_rotary(rotary, D, num_tokens)) return rc;
  if (kv_norm != nullptr) {
    if (const int rc = check_head_norm(kv_norm, 1)) return rc;
    WKV_CHECK_ARG(kv_norm->q_weight == nullptr, "kv_norm norms the compressed entries alone (k_weight)");
    WKV_CHECK_ARG(kv_norm->k_weight == nullptr || aligned16(kv_norm->k_weight), "the norm's weight must be 16-byte aligned");
  }
  if (num_tokens == 0) return WKV_OK;
  WKV_CHECK_ARG(slot_mapping != nullptr && reinterpret_cast<uintptr_t>(slot_mapping) % 8 == 0, "slot_mapping must be int64");
  if (const int rc = check_rows16(kv_c, kv_c_stride, 0, "kv_c")) return rc;
  if (const int rc = check_rows16(k_pe, k_pe_stride, 0, "k_pe")) return rc;
  WKV_CHECK_ARG(num_heads == 0 || (q_pe != nullptr && q_out != nullptr && reinterpret_cast<uintptr_t>(q_pe) % 2 == 0 &&
                    reinterpret_cast<uintptr_t>(q_out) % 2 == 0 && q_stride_t >= 0 && q_stride_h >= 0 &&
                    qo_stride_t >= 0 && qo_stride_h >= 0),
                "q_pe and its output must be non-NULL, aligned to their elements, their strides non-negative");
  const int half = rotary->rotary_dim / 2;
  const bool inter = rotary->interleaved != 0;
  Widths w(2, D, half, inter);
  if (num_heads > 0) {
    w.rows(q_pe, q_stride_t, q_stride_h);
    w.rows(q_out, qo_stride_t, qo_stride_h);
  }
  LatentArgs a{};
  a.q = HeadRows{q_pe, q_out, q_stride_t, q_stride_h, qo_stride_t, qo_stride_h};
  a.kvc = static_cast<const __bf16 *>(kv_c);
  a.kpe = static_cast<const __bf16 *>(k_pe);
  a.kvc_st = kv_c_stride;
  a.kpe_st = k_pe_stride;
  a.slots = slot_mapping;
  a.n = head_norm(kv_norm);
  a.a = angles(rotary);
  a.r = row_units(D, half, w.v);
  if (a.r.units > 64)
    return fail(WKV_ERR_UNSUPPORTED, "rope_dim %d with rotary_dim %d and rows of this alignment not supported", D, rotary->rotary_dim);
  a.tokens = num_tokens;
  a.heads = num_heads;
  a.rank = cache->kv_lora_rank;
  a.latent = static_cast<__bf16 *>(cache->latent);
  a.BS = cache->block_size;
  a.NB = cache->num_blocks;
  const RowGrid g(num_tokens, num_heads + 1, half, a.r.log_lanes);
  a.tile = g.tile;
  a.per = fast_div(g.per);
  a.last = fast_div(g.last);
  a.splits = fast_div(g.splits);
  a.row_wgs = g.wgs;
  const int64_t rest = (num_tokens + kWaves - 1) / kWaves;
  WKV_CHECK_ARG(a.row_wgs + rest <= INT32_MAX, "too many tokens and heads for one launch");
  const unsigned grid = static_cast<unsigned>(a.row_wgs + rest);
  const size_t lds = static_cast<size_t>(g.tile) * half * sizeof(float2);
  auto s = static_cast<hipStream_t>(stream);
  auto layout = [&](auto v) {
    constexpr int VV = decltype(v)::value;
    if (inter) mla_rotary_append_kernel<VV, true><<<grid, kThreads, lds, s>>>(a);
    else mla_rotary_append_kernel<VV, false><<<grid, kThreads, lds, s>>>(a);
  };
  if (w.v == 8) layout(std::integral_constant<int, 8>{});
  else if (w.v == 2) layout(std::integral_constant<int, 2>{});
  else layout(std::integral_constant<int, 1>{});
  WKV_CHECK_LAUNCH("mla_rotary_append");
  return WKV_OK;
}
