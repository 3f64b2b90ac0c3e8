// Keys and values into the paged cache with the norm of heads and the rotary
// positions on the way, and the queries to the attention, in one launch (gfx950).
// The mathematics of heads: norm_rotary_dev.h; the fp8 rule: kv_append_dev.h.
//
// The workgroups of a launch have one of three roles. Keys: of a bf16 cache as rows, several tokens a wave,
// so that the 16-byte pieces that it stores of a head lie together in the cache; of an fp8 cache run by run,
// because a block's scale follows from all of its new keys, coded from the registers in which they were
// normed and turned. Values: in bf16 a window of 64 tokens of one head, transposed through LDS (few tokens:
// an element at a time), in fp8 run by run. Queries: rows to rows. A latent cache has entries, a wave each,
// in the place of values, and its shared key is a kind of one head.
//
// Prompts are bound by HBM: 8 of 2,048 tokens, 32/8 heads of 128, bf16: 79 us for 403 MB, 5.1 TB/s, as a
// large copy (norm_rotary and append in turn: 65 + 34). Into fp8 blocks of 16, 8,386 tokens of 28/4 heads take 37,
// of which the queries alone are 27: a run's keys are a chain of round trips (slots, rows and positions, scale)
// of 6.5 us in a wave, so the workgroups of keys and values come first and the queries' fill the chip beside
// them (36.1 so, 41.1 behind them). Few tokens are bound by the launch and that chain (64 tokens bf16: 5.0
// us; 5 tokens fp8: 6.3).
//
// Larger fp8 blocks have longer runs, one wave each, whose pieces of 16 tokens follow each other and are normed and
// turned twice: those 8,386 tokens take 42, 58, 94 and 154 us in blocks of 32, 64, 128 and 256 (norm_rotary or
// apply_rotary and append in turn: 64, 71, 99, 150), and 16,384 tokens of 32/8 heads 97, 226 and 632 in blocks of 16,
// 64 and 256 (in turn 88, 164, 471).
#include <type_traits>

#include "kv_append_dev.h"
#include "norm_rotary_dev.h"

namespace wkv {

constexpr int kThreads = 256, kWaves = kThreads / 64;

// A cache's slots as blocks and offsets.
struct Slots {
  const int64_t *of;  // each token's
  int64_t count;      // slots of the cache
  FastDiv block;
  // Whether there is such a slot. Caches of 2^31 slots and more divide in 64 bits.
  __device__ __forceinline__ bool at(int64_t token, int64_t &blk, int &off) const {
    const int64_t slot = of[token];
    const bool there = slot >= 0 && slot < count;
    if (count <= INT32_MAX) {  // uniform
      const int s = there ? static_cast<int>(slot) : 0, b = s / block;
      blk = b;
      off = s - b * block.d;
    } else {
      blk = there ? slot / block.d : 0;
      off = there ? static_cast<int>(slot - blk * block.d) : 0;
    }
    return there;
  }
};

struct AppendArgs {
  Kind q, k;         // q.s.y: the queries' result; k.s.x: the keys
  int k_wgs, v_wgs;  // workgroups of keys, and of values; queries behind them
  const uint16_t *key, *val;
  int64_t kst, ksh, vst, vsh;
  Slots slots;
  HeadNorm n;
  Angles a;
  RowUnits r;
  int64_t tokens;
  int Hk;
  void *kc, *vc;
  float *ks, *vs;
  int BS;
  int window;  // tokens of a workgroup of values (and of fp8 keys)
};

// Queries to rows (K false), or keys to a bf16 cache.
template <int V, bool INTER, bool EACH, bool K, int LL, bool FAR>
__device__ __forceinline__ void heads_role(const AppendArgs &a, const Kind &k, int wg, float2 *turns) {
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const WaveTile w = wave_tile(k, a.r, a.tokens, wg, wave);
  if (w.tokens == 0) return;  // a whole wave; nothing below waits for another
  float2 *turn = turns + (wave << k.log_tg) * a.r.half;
  const void *weight = k.w;
  if (EACH && weight != nullptr) weight = static_cast<const char *>(weight) + w.h0 * k.ws * (a.n.wide ? 4 : 2);
  const int64_t t = w.t0 + w.t;
  HeadsOf<__bf16> of{static_cast<const __bf16 *>(k.s.x) + t * k.s.xt + w.h0 * k.s.xh, k.s.xh, nullptr, 0, 0, weight, k.ws};
  bool there = w.there;
  if (K) {
    int64_t blk;
    int off;
    there = a.slots.at(t, blk, off) && there;
    of.yh = static_cast<int64_t>(a.r.D) * a.BS;
    of.y = static_cast<__bf16 *>(a.kc) + (blk * a.Hk + w.h0) * of.yh + off * 8;  // (not used where there is no such block)
    of.piece = a.BS * 8;
  } else {
    of.y = static_cast<__bf16 *>(k.s.y) + t * k.s.yt + w.h0 * k.s.yh;
    of.yh = k.s.yh;
  }
  norm_turn_heads<__bf16, V, INTER, 1, FAR, K, EACH, LL>(
      a.r, a.n, turn + w.t * a.r.half, there, w.group, (64 >> a.r.log_lanes) >> k.log_tg, w.heads, of,
      [&] { wave_angles<K ? 2 : 1>(a.a, w.t0, w.tokens, turn); });
}

// ---------------------------------------------------------------------------
// bf16 values.
constexpr int kValueWindow = 64;
constexpr int64_t kValueWindowTokens = 256;  // below this the values go element by element, over more workgroups

template <int D>
__device__ __forceinline__ void values_role(const AppendArgs &a, int wg, uint8_t *lds) {
  constexpr int C = D / 8;
  uint16_t *vc = static_cast<uint16_t *>(a.vc);
  if (a.window == 1) {  // an item a thread: 8 elements of a token's head
    const int64_t i = static_cast<int64_t>(wg) * kThreads + threadIdx.x;
    if (i >= a.tokens * a.Hk * C) return;
    const int c = static_cast<int>(i % C);
    const int64_t th = i / C;
    const int h = static_cast<int>(th % a.Hk);
    const int64_t t = th / a.Hk;
    int64_t blk;
    int off;
    if (!a.slots.at(t, blk, off)) return;
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
  int64_t *place = reinterpret_cast<int64_t *>(lds + kValueWindow * RP);  // of a token's first value in the cache, -1: none
  int *whole = reinterpret_cast<int *>(place + kValueWindow);             // groups that are one run
  const int w = wg / a.Hk, h = wg - w * a.Hk, tid = threadIdx.x;
  const int64_t t0 = static_cast<int64_t>(w) * kValueWindow;
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
  if (tid < kValueWindow) {  // wave 0
    int64_t blk = 0, slot = -1;
    int off = 0;
    bool there = false;
    if (t0 + tid < a.tokens) {
      slot = a.slots.of[t0 + tid];
      there = a.slots.at(t0 + tid, blk, off);
    }
    place[tid] = there ? (blk * a.Hk + h) * D * a.BS + off : -1;
    const int64_t first = __shfl(slot, tid & ~7, 64);
    const uint64_t runs = __ballot(there && first % 8 == 0 && slot == first + (tid & 7));  // (blocks are multiples of 16)
    if ((tid & 7) == 0) whole[tid / 8] = ((runs >> tid) & 0xffu) == 0xffu;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < NG * D / kThreads; ++k) {
    const int i = tid + kThreads * k;
    const int g = 2 * (i / (2 * D)) + (i & 1), d = (i >> 1) % D;
    if (whole[g]) {
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = *reinterpret_cast<const uint16_t *>(lds + (8 * g + 2 * j) * RP + 2 * d);
        const uint32_t hi = *reinterpret_cast<const uint16_t *>(lds + (8 * g + 2 * j + 1) * RP + 2 * d);
        o[j] = lo | (hi << 16);
      }
      *reinterpret_cast<u32x4 *>(vc + place[8 * g] + static_cast<int64_t>(d) * a.BS) = u32x4{o[0], o[1], o[2], o[3]};
    } else {
      for (int j = 0; j < 8; ++j) {
        const int t = 8 * g + j;
        if (place[t] >= 0) vc[place[t] + static_cast<int64_t>(d) * a.BS] = *reinterpret_cast<const uint16_t *>(lds + t * RP + 2 * d);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// fp8 keys and values.
constexpr int kPiece = 16;  // tokens of a run taken at a time

// Codes of bf16 bits times inv, by the hardware's conversion; a NaN, which that codes with a sign of its own,
// as 0x7f and the NaN's sign.
struct Coder {
  float inv;
  bool any_nan;
  __device__ __forceinline__ u32x2 eight(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) const {
    u32x2 c = e4m3_pack8(w0, w1, w2, w3, inv);
    if (any_nan) {  // uniform
      const uint32_t w[4] = {w0, w1, w2, w3};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t b = (w[i >> 1] >> (16 * (i & 1))) & 0xffffu, at = 8 * (i & 3);
        if ((b & 0x7fffu) > 0x7f80u) c[i >> 2] = (c[i >> 2] & ~(0xffu << at)) | ((0x7fu | (b >> 8 & 0x80u)) << at);
      }
    }
    return c;
  }
  __device__ __forceinline__ uint32_t two(uint32_t w) const { return eight(w, 0u, 0u, 0u)[0]; }  // (and those of zeros)
};

// The largest magnitude of bf16 pairs, as bits: the two halves side by side; a NaN's are above infinity's.
struct Largest {
  typedef __attribute__((__vector_size__(4))) uint16_t u16x2;
  u16x2 top = {0, 0};
  __device__ __forceinline__ void pair(uint32_t w) {
    const u16x2 x = __builtin_bit_cast(u16x2, w & 0x7fff7fffu);
    top = __builtin_elementwise_max(top, x);
  }
  __device__ __forceinline__ uint32_t of_lane() const { return max(static_cast<uint32_t>(top[0]), static_cast<uint32_t>(top[1])); }
};

// 1 / s of a run's scale, a power of two in [2^-42, 2^120].
__device__ __forceinline__ float pow2_inverse(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
  return wave_reduce(v, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
}

// A pair's larger magnitude where a NaN counts as none.
__device__ __forceinline__ uint32_t without_nan(uint32_t w) {
  const uint32_t lo = w & 0x7fffu, hi = (w >> 16) & 0x7fffu;
  return max(lo > 0x7f80u ? 0u : lo, hi > 0x7f80u ? 0u : hi);
}

// A run's scale: its own, or where it does not begin the block the block's, grown if it is smaller, what the block
// held before coded again. The wave stores it.
template <int D, bool IS_V>
__device__ __forceinline__ float run_scale(uint8_t *codes, float *scales, int64_t blk, int h, int H, int BS, int first,
                                           float old, float amax) {
  float s = pow2_scale(amax);
  if (first != 0) {
    if (s > old)
      fp8_reencode_block<D, IS_V, true>(codes, blk, h, H, BS, first, old / s);
    else
      s = old;
  }
  if ((threadIdx.x & 63) == 0) scales[blk * H + h] = s;
  return s;
}

// The keys of head h of a run (r tokens from t on in block blk, the first at offset `first`), by a wave: as
// many tokens as it has groups side by side, the codes stored from where the heads were normed and turned, 8
// bytes a lane's run. Every wave of the workgroup calls it (a piece's angles are the workgroup's); active:
// the wave has a head. More than 16 tokens are normed and turned twice, for the scale and for the codes.
template <int D, int V, bool INTER, int LL>
__device__ __forceinline__ void append_keys(const AppendArgs &a, float2 *turn, int64_t t, int r, int64_t blk, int first,
                                            int h, bool active) {
  typedef typename VecOf<__bf16, V>::type Vec;
  constexpr int G = 64 >> LL, P = kPiece / G, W = V == 8 ? 4 : 1;
  static_assert(P * G == kPiece && (V == 8 || V == 2 || V == 1), "rows of a piece");
  uint8_t *kc = static_cast<uint8_t *>(a.kc);
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // (nothing that depends on it is held across the runs: registers)
  const int group = lane >> LL, u = lane & ((1 << LL) - 1), H = a.Hk, BS = a.BS;
  const bool all = 2 * a.r.half == D;
  int e0, e1;
  unit_runs<V, INTER>(a.r, u, e0, e1);
  float old = 0.f, w0[V], w1[V];
  if (active) {
    if (first != 0) old = a.ks[blk * H + h];
    load_weights<__bf16, V>(a.n, a.n.kw, h * a.n.kws + e0, w0);
    load_weights<__bf16, V>(a.n, a.n.kw, h * a.n.kws + e1, w1);
  }
  uint32_t k0[P][W], k1[P][W];
  int off[P];
  auto load = [&](int p0) __attribute__((always_inline)) {
    const int n = r - p0 < kPiece ? r - p0 : kPiece;
    Vec x0[P], x1[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int i = p * G + group;
      x0[p] = x1[p] = Vec{};
      off[p] = -1;
      if (active && i < n) {
        const __bf16 *x = reinterpret_cast<const __bf16 *>(a.key) + (t + p0 + i) * a.kst + h * a.ksh;
        x0[p] = *reinterpret_cast<const Vec *>(x + e0);
        x1[p] = *reinterpret_cast<const Vec *>(x + e1);
        off[p] = static_cast<int>(a.slots.of[t + p0 + i] - blk * BS);
      }
    }
    __syncthreads();  // the angles before have been read
    angles_of<4>(a.a, t + p0, n, threadIdx.x, kThreads, turn);
    __syncthreads();
    if (!active) return;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (p * G >= n) {  // uniform
#pragma unroll
        for (int i = 0; i < W; ++i) k0[p][i] = k1[p][i] = 0u;
        continue;
      }
      float f0[V], f1[V], ss = 0.f;
      widen<V, __bf16>(x0[p], f0);
      widen<V, __bf16>(x1[p], f1);
#pragma unroll
      for (int v = 0; v < V; ++v) ss = __builtin_fmaf(f0[v], f0[v], __builtin_fmaf(f1[v], f1[v], ss));
      ss = group_sum<LL>(ss, LL);
      const float inv = a.n.on ? __builtin_amdgcn_rsqf(__builtin_fmaf(ss, 1.f / static_cast<float>(D), a.n.eps)) : 1.f;
      unit_once<V, INTER>(turn + (off[p] >= 0 ? p * G + group : 0) * a.r.half, a.r.half, all, e0, e1, w0, w1, inv, f0, f1);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        k0[p][i] = V > 1 ? pack_bf16x2(f0[2 * i % V], f0[(2 * i + 1) % V]) : pack_bf16x2(f0[0], 0.f);
        k1[p][i] = V > 1 ? pack_bf16x2(f1[2 * i % V], f1[(2 * i + 1) % V]) : pack_bf16x2(f1[0], 0.f);
      }
      __builtin_amdgcn_sched_barrier(0);  // (a round's registers are free before the next one's are taken)
    }
  };
  Largest top;
  uint32_t finite = 0u;  // the largest without NaNs
  for (int p0 = 0; p0 < r; p0 += kPiece) {  // uniform
    load(p0);
    if (!active) continue;
    uint32_t here = 0u;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int i = 0; i < W; ++i) {
        k0[p][i] = off[p] >= 0 ? k0[p][i] : 0u;
        k1[p][i] = off[p] >= 0 ? k1[p][i] : 0u;
        top.pair(k0[p][i]);
        top.pair(k1[p][i]);
      }
    if (__any(top.of_lane() > 0x7f80u)) {
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < W; ++i) here = max(here, max(without_nan(k0[p][i]), without_nan(k1[p][i])));
    } else {
      here = top.of_lane();
    }
    finite = max(finite, here);
  }
  float s = 0.f;
  const uint32_t most = wave_max_bits(finite);
  if (active) s = run_scale<D, false>(kc, a.ks, blk, h, H, BS, first, old, __uint_as_float(most << 16));
  const Coder code{pow2_inverse(s), static_cast<bool>(__any(top.of_lane() > 0x7f80u))};
  for (int p0 = 0; p0 < r; p0 += kPiece) {
    if (r > kPiece) load(p0);
    if (!active) continue;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      uint8_t *y0 = kc + fp8_k_index<D>(blk, h, H, BS, off[p], e0), *y1 = kc + fp8_k_index<D>(blk, h, H, BS, off[p], e1);
      if constexpr (V == 8) {
        const u32x2 c0 = code.eight(k0[p][0], k0[p][1], k0[p][2], k0[p][3]);
        const u32x2 c1 = code.eight(k1[p][0], k1[p][1], k1[p][2], k1[p][3]);
        if (off[p] >= 0) {
          *reinterpret_cast<u32x2 *>(y0) = c0;
          *reinterpret_cast<u32x2 *>(y1) = c1;
        }
      } else if (off[p] >= 0) {
        typedef std::conditional_t<V == 2, uint16_t, uint8_t> Codes;
        *reinterpret_cast<Codes *>(y0) = static_cast<Codes>(code.two(k0[p][0]));
        *reinterpret_cast<Codes *>(y1) = static_cast<Codes>(code.two(k1[p][0]));
      }
    }
  }
}

// The values of head h of a run, by a wave: every lane has D / 64 of the d rows, and a byte of each for a token.
template <int D>
__device__ __forceinline__ void append_values(const AppendArgs &a, int64_t t, int r, int64_t blk, int first, int h) {
  constexpr int RV = D / 64;
  uint8_t *vc = static_cast<uint8_t *>(a.vc);
  const int lane = threadIdx.x & 63, m = lane & 15, H = a.Hk, BS = a.BS;
  const float old = first != 0 ? a.vs[blk * H + h] : 0.f;
  uint32_t vw[kPiece];
  int off = 0;  // offset in the block of the piece's token m
  auto load = [&](int p0) __attribute__((always_inline)) {
    const int n = r - p0 < kPiece ? r - p0 : kPiece, last = n - 1;
    if (n == 1) {  // uniform (a token a sequence)
      const uint16_t *p = a.val + (t + p0) * a.vst + h * a.vsh + RV * lane;
      vw[0] = RV == 2 ? *reinterpret_cast<const uint32_t *>(p) : *p;
#pragma unroll
      for (int i = 1; i < kPiece; ++i) vw[i] = vw[0];
    } else {
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        const uint16_t *p = a.val + (t + p0 + (i < last ? i : last)) * a.vst + h * a.vsh + RV * lane;
        if constexpr (RV == 2)
          vw[i] = *reinterpret_cast<const uint32_t *>(p);
        else
          vw[i] = *p;
      }
    }
    off = static_cast<int>(a.slots.of[t + p0 + (m < last ? m : last)] - blk * BS);
  };
  Largest top;
  uint32_t finite = 0u;
  for (int p0 = 0; p0 < r; p0 += kPiece) {  // uniform
    load(p0);
    uint32_t here = 0u;
#pragma unroll
    for (int i = 0; i < kPiece; ++i) top.pair(vw[i]);
    if (__any(top.of_lane() > 0x7f80u)) {
#pragma unroll
      for (int i = 0; i < kPiece; ++i) here = max(here, without_nan(vw[i]));
    } else {
      here = top.of_lane();
    }
    finite = max(finite, here);
  }
  const float s = run_scale<D, true>(vc, a.vs, blk, h, H, BS, first, old, __uint_as_float(wave_max_bits(finite) << 16));
  const Coder code{pow2_inverse(s), static_cast<bool>(__any(top.of_lane() > 0x7f80u))};
  for (int p0 = 0; p0 < r; p0 += kPiece) {
    if (r > kPiece) load(p0);
    const int n = r - p0 < kPiece ? r - p0 : kPiece;
    // consecutive offsets from a 16-aligned one on: a d row's 16 tokens in one store
    const int off0 = __builtin_amdgcn_readfirstlane(off);
    const bool whole = n == kPiece && off0 % kPiece == 0 && __all(off == off0 + m);
#pragma unroll
    for (int rr = 0; rr < RV; ++rr) {
      uint8_t *row = vc + fp8_v_index<D>(blk, h, H, BS, 0, RV * lane + rr);
      auto pair = [&](int i) { return ((vw[i] >> (16 * rr)) & 0xffffu) | (((vw[i + 1] >> (16 * rr)) & 0xffffu) << 16); };
      const u32x2 c0 = code.eight(pair(0), pair(2), pair(4), pair(6));
      const u32x2 c1 = code.eight(pair(8), pair(10), pair(12), pair(14));
      if (whole) {
        *reinterpret_cast<u32x4 *>(row + off0) = u32x4{c0[0], c0[1], c1[0], c1[1]};
      } else {
#pragma unroll
        for (int i = 0; i < kPiece; ++i)
          if (i < n) row[__builtin_amdgcn_readlane(off, i)] = static_cast<uint8_t>((i < 8 ? c0 : c1)[(i & 7) >> 2] >> (8 * (i & 3)));
      }
    }
  }
}

// The runs that begin in a window of the call's tokens, four heads a workgroup, one a wave: f(t, r, blk,
// first, h, active). The same in every wave.
template <class F>
__device__ __forceinline__ void window_runs(const AppendArgs &a, int wg, F f) {
  const int chunks = (a.Hk + kWaves - 1) / kWaves;
  const int w = wg / chunks;
  const int64_t t0 = static_cast<int64_t>(w) * a.window;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int h = (wg - w * chunks) * kWaves + wave;
  // lane l: token t0 - 1 + l, its block (-1: none); the window and, behind it, up to 63 - window tokens
  auto block_at = [&](int64_t tok) {
    int64_t blk;
    int off;
    return tok >= 0 && tok < a.tokens && a.slots.at(tok, blk, off) ? static_cast<int>(blk) : -1;
  };
  const int mine = block_at(t0 - 1 + lane);
  const int before = __shfl_up(mine, 1, 64);
  const uint64_t cont = __ballot(lane > 0 && mine >= 0 && mine == before);
  uint64_t starts = __ballot(lane > 0 && lane <= a.window && mine >= 0 && mine != before);
  while (starts != 0) {  // uniform
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
    f(t, r, static_cast<int64_t>(blk), static_cast<int>(a.slots.of[t] - static_cast<int64_t>(blk) * a.BS), h, h < a.Hk);
  }
}

// fp8: four waves a SIMD (128 registers, 60 bytes of them spilled at D = 128; 143 and three waves otherwise):
// 38.1 us in the place of 40.2 for 8,386 tokens of 28/4 heads.
template <int D, int V, bool INTER, bool FP8, bool EACH, bool FAR>
__global__ __launch_bounds__(kThreads, FP8 ? 4 : 1) void rotary_append_kernel(AppendArgs a) {
  constexpr int UNITS = D / (2 * V), LL = UNITS == 64 ? 6 : UNITS == 32 ? 5 : UNITS == 16 ? 4 : UNITS == 8 ? 3 : 2;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int wg = blockIdx.x;
  float2 *turn = reinterpret_cast<float2 *>(lds);
  if (wg < a.k_wgs) {
    if constexpr (FP8)
      window_runs(a, wg, [&](int64_t t, int r, int64_t blk, int first, int h, bool active) {
        append_keys<D, V, INTER, LL>(a, turn, t, r, blk, first, h, active);
      });
    else
      heads_role<V, INTER, EACH, true, LL, FAR>(a, a.k, wg, turn);
  } else if (wg < a.k_wgs + a.v_wgs) {
    if constexpr (FP8)
      window_runs(a, wg - a.k_wgs, [&](int64_t t, int r, int64_t blk, int first, int h, bool active) {
        if (active) append_values<D>(a, t, r, blk, first, h);
      });
    else
      values_role<D>(a, wg - a.k_wgs, lds);
  } else {
    heads_role<V, INTER, EACH, false, LL, FAR>(a, a.q, wg - a.k_wgs - a.v_wgs, turn);
  }
}

// ---------------------------------------------------------------------------
// The latent cache: rows of rope_dim (every query head's, and the shared key as a kind of its own), and the
// compressed entries, a wave each. 4,696 tokens of 128 heads of 64, each the end of a row of 192: 31 us by
// the trace, 36 a pass, where a copy of the same strided queries alone takes 34.
struct LatentArgs {
  Kind q, k;  // queries; the shared key, one head
  int entry_wgs, k_wgs;  // workgroups of entries, and of shared keys; queries behind them
  const __bf16 *kvc;
  int64_t kvc_st;
  Slots slots;
  HeadNorm n;  // of the entries: kw
  Angles a;
  RowUnits r;
  int64_t tokens;
  int rank;
  __bf16 *latent;
};

template <int V, bool INTER, int LL>
__global__ __launch_bounds__(kThreads) void mla_rotary_append_kernel(LatentArgs a) {
  extern __shared__ float2 turns[];
  const int width = a.rank + a.r.D;
  const int wg = static_cast<int>(blockIdx.x) - a.entry_wgs;
  if (wg >= 0) {
    const bool is_q = wg >= a.k_wgs;
    const Kind &k = is_q ? a.q : a.k;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const WaveTile w = wave_tile(k, a.r, a.tokens, is_q ? wg - a.k_wgs : wg, wave);
    if (w.tokens == 0) return;  // a whole wave; nothing below waits for another
    float2 *turn = turns + (wave << k.log_tg) * a.r.half;
    const int64_t t = w.t0 + w.t;
    HeadsOf<__bf16> of{static_cast<const __bf16 *>(k.s.x) + t * k.s.xt + w.h0 * k.s.xh, k.s.xh, nullptr, k.s.yh, 0, nullptr, 0};
    bool there = w.there;
    if (is_q) {
      of.y = static_cast<__bf16 *>(k.s.y) + t * k.s.yt + w.h0 * k.s.yh;
    } else {
      int64_t blk;
      int off;
      there = a.slots.at(t, blk, off) && there;
      of.y = a.latent + (blk * a.slots.block.d + off) * width + a.rank;
    }
    const HeadNorm none{};
    norm_turn_heads<__bf16, V, INTER, 1, false, false, false, LL>(
        a.r, none, turn + w.t * a.r.half, there, w.group, (64 >> a.r.log_lanes) >> k.log_tg, w.heads, of,
        [&] { wave_angles(a.a, w.t0, w.tokens, turn); });
    return;
  }
  const int lane = threadIdx.x & 63;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
  if (t >= a.tokens) return;  // a whole wave; nothing below waits for another
  int64_t blk;
  int off;
  if (!a.slots.at(t, blk, off)) return;
  typedef typename VecOf<__bf16, 8>::type Vec8;
  const __bf16 *x = a.kvc + t * a.kvc_st;
  __bf16 *y = a.latent + (blk * a.slots.block.d + off) * width;
  float f[8], ss = 0.f, inv = 1.f;
  if (a.n.on) {
    for (int e = 8 * lane; e < a.rank; e += 512) {
      widen<8, __bf16>(*reinterpret_cast<const Vec8 *>(x + e), f);
#pragma unroll
      for (int v = 0; v < 8; ++v) ss = __builtin_fmaf(f[v], f[v], ss);
    }
    inv = __builtin_amdgcn_rsqf(__builtin_fmaf(wave_sum(ss), 1.f / static_cast<float>(a.rank), a.n.eps));
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
  AppendArgs a{};
  a.key = static_cast<const uint16_t *>(key);
  a.val = static_cast<const uint16_t *>(value);
  a.kst = key_stride_t;
  a.ksh = key_stride_h;
  a.vst = value_stride_t;
  a.vsh = value_stride_h;
  a.slots = Slots{slot_mapping, cache->num_blocks * cache->block_size, fast_div(cache->block_size)};
  a.n = head_norm(norm);
  a.a = angles(rotary);
  a.r = row_units(D, half, w.v);
  a.tokens = num_tokens;
  a.Hk = Hk;
  a.kc = cache->k;
  a.vc = cache->v;
  a.ks = cache->k_scale;
  a.vs = cache->v_scale;
  a.BS = cache->block_size;
  const KindGrid gq(num_tokens, num_q_heads, a.r.log_lanes, false), gk(num_tokens, fp8 ? 0 : Hk, a.r.log_lanes, true);
  int64_t k_wgs = gk.wgs;
  a.q = Kind{HeadRows{q, q_out, q_stride_t, q_stride_h, qo_stride_t, qo_stride_h}, a.n.qw, a.n.qws, num_q_heads, gq.log_tg,
             gq.per, fast_div(gq.splits)};
  a.k = Kind{HeadRows{key, nullptr, key_stride_t, key_stride_h, 0, 0}, a.n.kw, a.n.kws, Hk, gk.log_tg, gk.per,
             fast_div(gk.splits)};
  const bool each = (a.n.qw != nullptr && a.n.qws != 0) || (a.n.kw != nullptr && a.n.kws != 0);
  size_t lds = (static_cast<size_t>(kWaves) << (gq.log_tg > gk.log_tg ? gq.log_tg : gk.log_tg)) * half * sizeof(float2);
  int64_t rest;
  if (fp8) {
    // a window of 16 tokens for prompts, whose runs mostly begin 16 apart; of one where every token may be a run
    a.window = num_tokens >= 4096 ? 16 : num_tokens >= 1024 ? 4 : 1;
    rest = (num_tokens + a.window - 1) / a.window * ((Hk + kWaves - 1) / kWaves);
    k_wgs = rest;
    const size_t need = static_cast<size_t>(kPiece) * half * sizeof(float2);
    lds = lds > need ? lds : need;
  } else if (num_tokens < kValueWindowTokens) {
    a.window = 1;
    rest = (num_tokens * Hk * (D / 8) + kThreads - 1) / kThreads;
  } else {
    a.window = kValueWindow;
    rest = (num_tokens + kValueWindow - 1) / kValueWindow * Hk;
    const size_t need = kValueWindow * (D * 2 + 8) + kValueWindow * sizeof(int64_t) + kValueWindow / 8 * sizeof(int);
    lds = lds > need ? lds : need;
  }
  WKV_CHECK_ARG(gq.wgs + k_wgs + rest <= kMaxWorkgroups, "too many tokens and heads for one launch");
  a.k_wgs = static_cast<int>(k_wgs);
  a.v_wgs = static_cast<int>(rest);
  const unsigned grid = static_cast<unsigned>(gq.wgs + k_wgs + rest);
  // Rows far larger than the caches go past them (8 prompts of 2,048 tokens, 32/8 heads of 128: 81 us, 88
  // near); the cache's keys and values stay, for the attention.
  const bool far = num_tokens * (num_q_heads + Hk) * D * 2 >= (64 << 20);
  auto s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto d, auto v, auto in) {
    constexpr int DD = decltype(d)::value, VV = decltype(v)::value;
    constexpr bool IN = decltype(in)::value;
    if constexpr (VV == 8) {
      if (far && fp8 && !each) return rotary_append_kernel<DD, VV, IN, true, false, true><<<grid, kThreads, lds, s>>>(a);
      if (far && !each) return rotary_append_kernel<DD, VV, IN, false, false, true><<<grid, kThreads, lds, s>>>(a);
    }
    if (fp8 && each) return rotary_append_kernel<DD, VV, IN, true, true, false><<<grid, kThreads, lds, s>>>(a);
    if (fp8) return rotary_append_kernel<DD, VV, IN, true, false, false><<<grid, kThreads, lds, s>>>(a);
    if (each) return rotary_append_kernel<DD, VV, IN, false, true, false><<<grid, kThreads, lds, s>>>(a);
    rotary_append_kernel<DD, VV, IN, false, false, false><<<grid, kThreads, lds, s>>>(a);
  };
  auto layout = [&](auto d, auto v) {
    if (inter) launch(d, v, std::true_type{}); else launch(d, v, std::false_type{});
  };
  auto width = [&](auto d) {
    if (w.v == 8) layout(d, std::integral_constant<int, 8>{});
    else if (w.v == 2) layout(d, std::integral_constant<int, 2>{});
    else layout(d, std::integral_constant<int, 1>{});
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
    WKV_CHECK_ARG(kv_norm->k_weight == nullptr || (aligned16(kv_norm->k_weight) && kv_norm->k_weight_stride_h == 0),
                  "the norm's weight must be one row of kv_lora_rank, 16-byte aligned");
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
  a.kvc = static_cast<const __bf16 *>(kv_c);
  a.kvc_st = kv_c_stride;
  a.slots = Slots{slot_mapping, cache->num_blocks * cache->block_size, fast_div(cache->block_size)};
  a.n = head_norm(kv_norm);
  a.a = angles(rotary);
  a.r = row_units(D, half, w.v);
  if (a.r.units > 64)
    return fail(WKV_ERR_UNSUPPORTED, "rope_dim %d with rotary_dim %d and rows of this alignment not supported", D, rotary->rotary_dim);
  a.tokens = num_tokens;
  a.rank = cache->kv_lora_rank;
  a.latent = static_cast<__bf16 *>(cache->latent);
  const KindGrid gq(num_tokens, num_heads, a.r.log_lanes, false), gk(num_tokens, 1, a.r.log_lanes, true);
  a.q = Kind{HeadRows{q_pe, q_out, q_stride_t, q_stride_h, qo_stride_t, qo_stride_h}, nullptr, 0, num_heads, gq.log_tg, gq.per,
             fast_div(gq.splits)};
  a.k = Kind{HeadRows{k_pe, nullptr, k_pe_stride, 0, 0, 0}, nullptr, 0, 1, gk.log_tg, gk.per, fast_div(gk.splits)};
  const int64_t rest = (num_tokens + kWaves - 1) / kWaves;
  WKV_CHECK_ARG(gq.wgs + gk.wgs + rest <= kMaxWorkgroups, "too many tokens and heads for one launch");
  a.entry_wgs = static_cast<int>(rest);
  a.k_wgs = static_cast<int>(gk.wgs);
  const unsigned grid = static_cast<unsigned>(gq.wgs + gk.wgs + rest);
  const size_t lds = (static_cast<size_t>(kWaves) << (gq.log_tg > gk.log_tg ? gq.log_tg : gk.log_tg)) * half * sizeof(float2);
  auto s = static_cast<hipStream_t>(stream);
  auto layout = [&](auto v) {
    constexpr int VV = decltype(v)::value;
    if constexpr (VV == 8) {  // rows of 64: their lanes as a constant
      if (a.r.log_lanes == 2 && inter) return mla_rotary_append_kernel<VV, true, 2><<<grid, kThreads, lds, s>>>(a);
      if (a.r.log_lanes == 2) return mla_rotary_append_kernel<VV, false, 2><<<grid, kThreads, lds, s>>>(a);
    }
    if (inter) mla_rotary_append_kernel<VV, true, -1><<<grid, kThreads, lds, s>>>(a);
    else mla_rotary_append_kernel<VV, false, -1><<<grid, kThreads, lds, s>>>(a);
  };
  if (w.v == 8) layout(std::integral_constant<int, 8>{});
  else if (w.v == 2) layout(std::integral_constant<int, 2>{});
  else layout(std::integral_constant<int, 1>{});
  WKV_CHECK_LAUNCH("mla_rotary_append");
  return WKV_OK;
}
