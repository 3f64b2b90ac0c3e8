// Norms of queries and keys for each head with the rotary positions in the same
// pass, forward and backward (gfx950). The mathematics: norm_rotary_dev.h.
//
// Forward: a wave takes a token and some or all of its queries or keys. Bound by HBM for prompts: 16,384
// tokens of 40 heads of 128, bf16, 64 us, 5.2 TB/s, the rate of a large copy (two tokens a wave 69, eight,
// each lane group its own, 81: the heads of a token lie together); by the launch and two round trips for a
// token (3.6-4.0 us).
//
// Backward, from the inputs and the outputs' gradient g: with z = R^T g, m = z (w + offset), r the
// reciprocal root mean square,
//   dx = r (m - x r^2 mean(m x)),   dw = sum over rows of z x r.
// A group of lanes keeps its elements of dw in registers over all the rows that it takes; workgroups leave
// their sums in the workspace, and a second kernel adds them up, in an order that the sizes alone give. Bound by
// HBM: 16,384 tokens of 40 heads of 128, bf16, 98 us (503 MB, 5.1 TB/s) and 5 for the sums; 8,191 tokens of 24 heads 36
// (151 MB, 4.2 TB/s) and 4 for the sums.
#include <algorithm>
#include <type_traits>

#include "norm_rotary_dev.h"

namespace wkv {

constexpr int kNormThreads = 256, kNormWaves = kNormThreads / 64;

struct NormRotaryArgs {
  Kind q, k;
  HeadNorm n;
  Angles a;
  RowUnits r;
  int64_t tokens;
  int q_wgs;  // workgroups that take queries; keys behind them
};

template <class T, int V, bool INTER, int U, bool FAR, bool EACH, int LL>
__global__ __launch_bounds__(kNormThreads) void norm_rotary_kernel(NormRotaryArgs a) {
  extern __shared__ float2 turns[];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const bool is_q = static_cast<int>(blockIdx.x) < a.q_wgs;
  const Kind &k = is_q ? a.q : a.k;
  const WaveTile w = wave_tile(k, a.r, a.tokens, is_q ? blockIdx.x : blockIdx.x - a.q_wgs, wave);
  if (w.tokens == 0) return;  // a whole wave; nothing below waits for another
  float2 *turn = turns + (wave << k.log_tg) * a.r.half;
  const void *weight = k.w;
  if (EACH && weight != nullptr) weight = static_cast<const char *>(weight) + w.h0 * k.ws * (a.n.wide ? 4 : sizeof(T));
  const int64_t t = w.t0 + w.t;
  const HeadsOf<T> of{static_cast<const T *>(k.s.x) + t * k.s.xt + w.h0 * k.s.xh, k.s.xh,
                      static_cast<T *>(k.s.y) + t * k.s.yt + w.h0 * k.s.yh, k.s.yh, 0, weight, k.ws};
  norm_turn_heads<T, V, INTER, U, FAR, false, EACH, LL>(
      a.r, a.n, turn + w.t * a.r.half, w.there, w.group, (64 >> a.r.log_lanes) >> k.log_tg, w.heads, of,
      [&] { wave_angles(a.a, w.t0, w.tokens, turn); });
}

// ---------------------------------------------------------------------------
// Backward.
struct GradRows {
  const void *x, *g;
  void *dx;  // nullptr: not asked for
  int64_t xt, xh, gt, gh, dt, dh;
};

// A kind's workgroups: `wgs` along the tokens for each of its ranges of heads. split: a range is as many heads as
// a wave has groups, and every group keeps to one (also where each head has a weight of its own); else it is
// all heads, which every wave's groups walk for some tokens.
struct GradKind {
  GradRows s;
  const void *w;
  int64_t ws;
  int heads, each, split, ranges, wgs;
  int log_tg;
  int64_t first;  // of its sums in the workspace, in rows of D
};

struct NormGradArgs {
  GradKind q, k;
  HeadNorm n;
  Angles a;  // sign: the transpose's
  RowUnits r;
  int64_t tokens;
  float *partial;  // [wgs][heads][D], or [ranges][wgs][D], of queries, then keys; nullptr: no weight's gradient
};

template <class T, int V, bool INTER, int U, bool FAR, bool DW, int LL>
__global__ __launch_bounds__(kNormThreads) void norm_rotary_grad_kernel(NormGradArgs a) {
  typedef typename VecOf<T, V>::type Vec;
  extern __shared__ float2 turns[];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int nq = a.q.ranges * a.q.wgs;
  const bool is_q = static_cast<int>(blockIdx.x) < nq;
  const GradKind &k = is_q ? a.q : a.k;
  const int b = is_q ? blockIdx.x : blockIdx.x - nq;
  const int range = b / k.wgs, wg = b - range * k.wgs;
  const int log_lanes = LL >= 0 ? LL : a.r.log_lanes;
  const int lanes = 1 << log_lanes, u0 = threadIdx.x & (lanes - 1), g = (threadIdx.x & 63) >> log_lanes;
  const int groups = 64 >> log_lanes, tg = 1 << k.log_tg, step = k.split ? groups : groups >> k.log_tg;
  const int h0 = range * (k.split ? groups : k.heads), heads = k.split ? (k.heads - h0 < groups ? k.heads - h0 : groups) : k.heads;
  const int t = k.split ? 0 : g & (tg - 1), first = k.split ? g : g >> k.log_tg;
  const int rounds = k.split ? tg : (heads + step - 1) / step;
  float2 *turn = turns + (wave << k.log_tg) * a.r.half;
  const float inv_d = 1.f / static_cast<float>(a.r.D);
  const bool all = 2 * a.r.half == a.r.D;
  int e0[U], e1[U];
  bool mine[U];
  float w0[U][V], w1[U][V], acc0[U][V], acc1[U][V];
#pragma unroll
  for (int j = 0; j < U; ++j) {
    const int u = u0 + lanes * j;
    mine[j] = u < a.r.units;
    e0[j] = e1[j] = 0;
    if (mine[j]) unit_runs<V, INTER>(a.r, u, e0[j], e1[j]);
    const int64_t wh = k.each && first < heads ? (h0 + first) * k.ws : 0;
    load_weights<T, V>(a.n, k.w, wh + e0[j], w0[j]);
    load_weights<T, V>(a.n, k.w, wh + e1[j], w1[j]);
#pragma unroll
    for (int v = 0; v < V; ++v) acc0[j][v] = acc1[j][v] = 0.f;
  }
  // A round is the wave's tokens of a block and `step` heads (split: one of the tokens and the range's heads); the
  // next one's loads are in flight over it.
  const int64_t blocks = ((a.tokens - 1) >> k.log_tg) + 1, stride = static_cast<int64_t>(k.wgs) * kNormWaves;
  Vec nx0[U], nx1[U], ng0[U], ng1[U];
  auto load = [&](int64_t block, int round) __attribute__((always_inline)) {
    const int64_t tt = (block << k.log_tg) + (k.split ? round : t);
    const int h = (k.split ? 0 : round * step) + first;
    const T *x = static_cast<const T *>(k.s.x) + tt * k.s.xt + (h0 + h) * k.s.xh;
    const T *gr = static_cast<const T *>(k.s.g) + tt * k.s.gt + (h0 + h) * k.s.gh;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      nx0[j] = nx1[j] = ng0[j] = ng1[j] = Vec{};
      if (mine[j] && tt < a.tokens && h < heads) {
        const Vec *px0 = reinterpret_cast<const Vec *>(x + e0[j]), *px1 = reinterpret_cast<const Vec *>(x + e1[j]);
        const Vec *pg0 = reinterpret_cast<const Vec *>(gr + e0[j]), *pg1 = reinterpret_cast<const Vec *>(gr + e1[j]);
        nx0[j] = FAR ? __builtin_nontemporal_load(px0) : *px0;
        nx1[j] = FAR ? __builtin_nontemporal_load(px1) : *px1;
        ng0[j] = FAR ? __builtin_nontemporal_load(pg0) : *pg0;
        ng1[j] = FAR ? __builtin_nontemporal_load(pg1) : *pg1;
      }
    }
  };
  UnitTurn<V> turned[U];
  int64_t block = static_cast<int64_t>(wg) * kNormWaves + wave;
  int round = 0;
  if (block < blocks) load(block, 0);
  while (block < blocks) {  // uniform
    Vec x0[U], x1[U], g0[U], g1[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      x0[j] = nx0[j];
      x1[j] = nx1[j];
      g0[j] = ng0[j];
      g1[j] = ng1[j];
    }
    const int64_t this_block = block;
    const int this_round = round;
    if (++round == rounds) {
      round = 0;
      block += stride;
    }
    if (block < blocks) load(block, round);
    const int64_t t0 = this_block << k.log_tg;
    const int nt = a.tokens - t0 < tg ? static_cast<int>(a.tokens - t0) : tg;
    const int mt = k.split ? this_round : t;  // the lane's token of the block
    if (this_round == 0) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the block before has been read
      __builtin_amdgcn_wave_barrier();
      wave_angles(a.a, t0, nt, turn);
    }
    if (this_round == 0 || k.split) {
#pragma unroll
      for (int j = 0; j < U; ++j)
        unit_turn<V, INTER>(turn + (mt < nt ? mt : 0) * a.r.half, a.r.half, all, e0[j], e1[j], turned[j]);
    }
    float f0[U][V], f1[U][V], z0[U][V], z1[U][V], ss = 0.f, sm = 0.f;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      widen<V, T>(x0[j], f0[j]);
      widen<V, T>(x1[j], f1[j]);
      widen<V, T>(g0[j], z0[j]);
      widen<V, T>(g1[j], z1[j]);
      unit_back<V, INTER>(turned[j], all, z0[j], z1[j]);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        ss = __builtin_fmaf(f0[j][v], f0[j][v], __builtin_fmaf(f1[j][v], f1[j][v], ss));
        sm = __builtin_fmaf(z0[j][v] * w0[j][v], f0[j][v], __builtin_fmaf(z1[j][v] * w1[j][v], f1[j][v], sm));
      }
    }
    ss = group_sum<LL>(ss, log_lanes);
    sm = group_sum<LL>(sm, log_lanes);
    const float inv = __builtin_amdgcn_rsqf(__builtin_fmaf(ss, inv_d, a.n.eps));
    const float back = sm * inv_d * inv * inv;
    const int64_t tt = t0 + mt;
    const int h = (k.split ? 0 : this_round * step) + first;
    const bool store = k.s.dx != nullptr && tt < a.tokens && h < heads;
    T *y = static_cast<T *>(k.s.dx) + tt * k.s.dt + (h0 + h) * k.s.dh;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      Vec o0, o1;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (DW) {
          acc0[j][v] = __builtin_fmaf(z0[j][v], f0[j][v] * inv, acc0[j][v]);
          acc1[j][v] = __builtin_fmaf(z1[j][v], f1[j][v] * inv, acc1[j][v]);
        }
        o0[v] = static_cast<T>(inv * __builtin_fmaf(-back, f0[j][v], z0[j][v] * w0[j][v]));
        o1[v] = static_cast<T>(inv * __builtin_fmaf(-back, f1[j][v], z1[j][v] * w1[j][v]));
      }
      if (store && mine[j]) {
        Vec *p0 = reinterpret_cast<Vec *>(y + e0[j]), *p1 = reinterpret_cast<Vec *>(y + e1[j]);
        if (FAR) {
          __builtin_nontemporal_store(o0, p0);
          __builtin_nontemporal_store(o1, p1);
        } else {
          *p0 = o0;
          *p1 = o1;
        }
      }
    }
  }
  if (!DW) return;
  // The sums: of a wave's groups by butterflies (one weight for all heads), of the waves through LDS.
  float *sums = reinterpret_cast<float *>(turns);  // [waves][rows][D]
  const int rows = k.each ? groups : 1;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < U; ++j) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float s0 = acc0[j][v], s1 = acc1[j][v];
      if (!k.each)
        for (int o = lanes; o < 64; o *= 2) {  // uniform
          s0 += __shfl_xor(s0, o, 64);
          s1 += __shfl_xor(s1, o, 64);
        }
      if (mine[j] && g < rows) {
        sums[(wave * rows + g) * a.r.D + e0[j] + v] = s0;
        sums[(wave * rows + g) * a.r.D + e1[j] + v] = s1;
      }
    }
  }
  __syncthreads();
  const int n = k.each ? heads : 1;  // a group's number is its head's, one token a wave
  float *out = a.partial + (k.first + (k.each ? static_cast<int64_t>(wg) * k.heads + h0 : b)) * a.r.D;
  for (int d = threadIdx.x; d < n * a.r.D; d += kNormThreads) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kNormWaves; ++i) s += sums[i * rows * a.r.D + d];
    out[d] = s;
  }
}

// The weights' gradients from the workgroups' sums: a workgroup adds up 64
// elements of one head's row, a sixteenth of the sums each wave.
constexpr int kSumWaves = 16;
struct WeightGrads {
  const float *partial;
  void *dq, *dk;  // nullptr: not asked for
  int q_rows, k_rows, q_wgs, k_wgs, D;
  int dtype;  // of the gradients: 0 fp32, 1 bf16, 2 fp16
};

__global__ __launch_bounds__(64 * kSumWaves) void norm_weight_grad_kernel(WeightGrads a) {
  __shared__ float sums[kSumWaves][64];
  const bool is_q = static_cast<int>(blockIdx.x) < a.q_rows;
  const int row = is_q ? blockIdx.x : blockIdx.x - a.q_rows;
  void *out = is_q ? a.dq : a.dk;
  if (out == nullptr) return;  // uniform
  const int n = is_q ? a.q_wgs : a.k_wgs;
  const int64_t rows = is_q ? a.q_rows : a.k_rows;
  const float *p = a.partial + ((is_q ? 0 : static_cast<int64_t>(a.q_rows) * a.q_wgs) + row) * a.D;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, d = blockIdx.y * 64 + lane;
  float s = 0.f;
  if (d < a.D) {
#pragma unroll 8
    for (int i = wave; i < n; i += kSumWaves) s += p[i * rows * a.D + d];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || d >= a.D) return;
#pragma unroll
  for (int i = 1; i < kSumWaves; ++i) s += sums[i][lane];
  const int64_t at = static_cast<int64_t>(row) * a.D + d;
  if (a.dtype == 0)
    static_cast<float *>(out)[at] = s;
  else if (a.dtype == 1)
    static_cast<__bf16 *>(out)[at] = static_cast<__bf16>(s);
  else
    static_cast<_Float16 *>(out)[at] = static_cast<_Float16>(s);
}

// ---------------------------------------------------------------------------
// Host. The launches. Heads of 64 and 128 in 16-byte accesses have their lanes as a constant (16,384 tokens of 40
// heads of 128, bf16: 65.6 us forward, 66.0 without, and 70.9 and 72.1 with each head's weights; forward and backward
// 166.4 and 168.9).
template <class T, int V, bool INTER, bool EACH>
static void launch_norm(const NormRotaryArgs &a, bool far, unsigned grid, size_t lds, hipStream_t s) {
  if (a.r.units > 64) {
    if constexpr (V <= 2) norm_rotary_kernel<T, V, INTER, 4, false, EACH, -1><<<grid, kNormThreads, lds, s>>>(a);
    return;
  }
  if constexpr (V * sizeof(T) == 16) {
    constexpr int L64 = sizeof(T) == 2 ? 2 : 3, L128 = L64 + 1;
    if (a.r.log_lanes == L128 && far) return norm_rotary_kernel<T, V, INTER, 1, true, EACH, L128><<<grid, kNormThreads, lds, s>>>(a);
    if (a.r.log_lanes == L128) return norm_rotary_kernel<T, V, INTER, 1, false, EACH, L128><<<grid, kNormThreads, lds, s>>>(a);
    if (a.r.log_lanes == L64 && far) return norm_rotary_kernel<T, V, INTER, 1, true, EACH, L64><<<grid, kNormThreads, lds, s>>>(a);
    if (a.r.log_lanes == L64) return norm_rotary_kernel<T, V, INTER, 1, false, EACH, L64><<<grid, kNormThreads, lds, s>>>(a);
  }
  norm_rotary_kernel<T, V, INTER, 1, false, EACH, -1><<<grid, kNormThreads, lds, s>>>(a);
}

template <class T, int V, bool INTER, bool DW>
static void launch_norm_grad(const NormGradArgs &a, bool far, unsigned grid, size_t lds, hipStream_t s) {
  if (a.r.units > 64) {
    if constexpr (V <= 2) norm_rotary_grad_kernel<T, V, INTER, 4, false, DW, -1><<<grid, kNormThreads, lds, s>>>(a);
    return;
  }
  if constexpr (V * sizeof(T) == 16) {
    constexpr int L64 = sizeof(T) == 2 ? 2 : 3, L128 = L64 + 1;
    if (a.r.log_lanes == L128 && far) return norm_rotary_grad_kernel<T, V, INTER, 1, true, DW, L128><<<grid, kNormThreads, lds, s>>>(a);
    if (a.r.log_lanes == L128) return norm_rotary_grad_kernel<T, V, INTER, 1, false, DW, L128><<<grid, kNormThreads, lds, s>>>(a);
    if (a.r.log_lanes == L64 && far) return norm_rotary_grad_kernel<T, V, INTER, 1, true, DW, L64><<<grid, kNormThreads, lds, s>>>(a);
    if (a.r.log_lanes == L64) return norm_rotary_grad_kernel<T, V, INTER, 1, false, DW, L64><<<grid, kNormThreads, lds, s>>>(a);
    if (far) return norm_rotary_grad_kernel<T, V, INTER, 1, true, DW, -1><<<grid, kNormThreads, lds, s>>>(a);
  }
  norm_rotary_grad_kernel<T, V, INTER, 1, false, DW, -1><<<grid, kNormThreads, lds, s>>>(a);
}

// f(element type's zero, width, layout) for the call's.
template <class F>
static void with_types(int dtype, int v, bool inter, F f) {
  auto width = [&](auto zero) {
    using T = decltype(zero);
    constexpr int W = 16 / sizeof(T);
    auto layout = [&](auto vv) {
      if (inter) f(zero, vv, std::true_type{}); else f(zero, vv, std::false_type{});
    };
    if (v == W) layout(std::integral_constant<int, W>{});
    else if (v == 2) layout(std::integral_constant<int, 2>{});
    else layout(std::integral_constant<int, 1>{});
  };
  if (dtype == 0) width(0.f);
  else if (dtype == 1) width(static_cast<__bf16>(0.f));
  else width(static_cast<_Float16>(0.f));
}

}  // namespace wkv

using namespace wkv;

namespace {

int check_norm_call(int32_t dtype, int32_t num_q_heads, int32_t num_k_heads, int32_t head_dim,
                    const wkv_head_norm_t *norm, const wkv_rotary_t *rotary, int64_t num_tokens) {
  WKV_CHECK_ARG(dtype >= 0 && dtype <= 2, "dtype must be 0 (fp32), 1 (bf16) or 2 (fp16) (got %d)", dtype);
  WKV_CHECK_ARG(num_tokens >= 0 && num_tokens <= INT32_MAX, "num_tokens must be in [0, 2^31) (got %lld)",
                (long long)num_tokens);
  WKV_CHECK_ARG(num_q_heads >= 0 && num_k_heads >= 0 && num_q_heads <= 65535 && num_k_heads <= 65535,
                "head counts must be in [0, 65535]");
  WKV_CHECK_ARG(head_dim > 0 && head_dim % 2 == 0 && head_dim <= WKV_ROTARY_MAX_DIM,
                "head_dim must be even and in [2, %d] (got %d)", WKV_ROTARY_MAX_DIM, head_dim);
  if (norm != nullptr) {
    const int rc = check_head_norm(norm, dtype);
    if (rc != WKV_OK) return rc;
  }
  return rotary == nullptr ? WKV_OK : check_rotary(rotary, head_dim, num_tokens);
}

bool rows_ok(const void *x, int64_t st, int64_t sh, int esz) {
  return x != nullptr && reinterpret_cast<uintptr_t>(x) % esz == 0 && st >= 0 && sh >= 0;
}

}  // namespace

// norm or rotary may be NULL, not both.
static int norm_rotary_call(int32_t dtype, const void *q, int64_t q_stride_t, int64_t q_stride_h, void *q_out,
                            int64_t qo_stride_t, int64_t qo_stride_h, int32_t num_q_heads, const void *k,
                            int64_t k_stride_t, int64_t k_stride_h, void *k_out, int64_t ko_stride_t,
                            int64_t ko_stride_h, int32_t num_k_heads, int32_t head_dim, const wkv_head_norm_t *norm,
                            const wkv_rotary_t *rotary, int64_t num_tokens, void *stream) {
  if (const int rc = check_norm_call(dtype, num_q_heads, num_k_heads, head_dim, norm, rotary, num_tokens)) return rc;
  const int H = num_q_heads + num_k_heads, esz = dtype == 0 ? 4 : 2;
  if (num_tokens == 0 || H == 0) return WKV_OK;
  WKV_CHECK_ARG((num_q_heads == 0 || (rows_ok(q, q_stride_t, q_stride_h, esz) && rows_ok(q_out, qo_stride_t, qo_stride_h, esz))) &&
                    (num_k_heads == 0 || (rows_ok(k, k_stride_t, k_stride_h, esz) && rows_ok(k_out, ko_stride_t, ko_stride_h, esz))),
                "q / k and their outputs must be non-NULL, aligned to their elements, their strides non-negative");
  const int half = rotary != nullptr ? rotary->rotary_dim / 2 : 0;
  const bool inter = rotary != nullptr && rotary->interleaved != 0;
  NormRotaryArgs a{};
  a.n = head_norm(norm);
  a.a = angles(rotary);
  a.tokens = num_tokens;
  Widths w(esz, head_dim, half, inter);
  const int wsz = a.n.wide ? 4 : 2;
  if (num_q_heads > 0) {
    w.rows(q, q_stride_t, q_stride_h);
    w.rows(q_out, qo_stride_t, qo_stride_h);
    w.weights(a.n.qw, a.n.qws, wsz);
  }
  if (num_k_heads > 0) {
    w.rows(k, k_stride_t, k_stride_h);
    w.rows(k_out, ko_stride_t, ko_stride_h);
    w.weights(a.n.kw, a.n.kws, wsz);
  }
  a.r = row_units(head_dim, half, w.v);
  const KindGrid gq(num_tokens, num_q_heads, a.r.log_lanes, false), gk(num_tokens, num_k_heads, a.r.log_lanes, false);
  a.q = Kind{HeadRows{q, q_out, q_stride_t, q_stride_h, qo_stride_t, qo_stride_h}, a.n.qw, a.n.qws, num_q_heads,
             gq.log_tg, gq.per, fast_div(gq.splits)};
  a.k = Kind{HeadRows{k, k_out, k_stride_t, k_stride_h, ko_stride_t, ko_stride_h}, a.n.kw, a.n.kws, num_k_heads,
             gk.log_tg, gk.per, fast_div(gk.splits)};
  WKV_CHECK_ARG(gq.wgs + gk.wgs <= kMaxWorkgroups, "too many tokens and heads for one launch");
  a.q_wgs = static_cast<int>(gq.wgs);
  const bool each = (a.n.qw != nullptr && a.n.qws != 0) || (a.n.kw != nullptr && a.n.kws != 0);
  const bool far = num_tokens * H * head_dim * esz >= (64 << 20);
  const unsigned grid = static_cast<unsigned>(gq.wgs + gk.wgs);
  const int log_tg = gq.log_tg > gk.log_tg ? gq.log_tg : gk.log_tg;
  const size_t lds = (static_cast<size_t>(kNormWaves) << log_tg) * half * sizeof(float2);
  auto s = static_cast<hipStream_t>(stream);
  with_types(dtype, w.v, inter, [&](auto zero, auto v, auto in) {
    using T = decltype(zero);
    if (each) launch_norm<T, decltype(v)::value, decltype(in)::value, true>(a, far, grid, lds, s);
    else launch_norm<T, decltype(v)::value, decltype(in)::value, false>(a, far, grid, lds, s);
  });
  WKV_CHECK_LAUNCH("norm_rotary");
  return WKV_OK;
}

extern "C" int wkv_norm_rotary(int32_t dtype, const void *q, int64_t q_stride_t, int64_t q_stride_h, void *q_out,
                               int64_t qo_stride_t, int64_t qo_stride_h, int32_t num_q_heads, const void *k,
                               int64_t k_stride_t, int64_t k_stride_h, void *k_out, int64_t ko_stride_t,
                               int64_t ko_stride_h, int32_t num_k_heads, int32_t head_dim,
                               const wkv_head_norm_t *norm, const wkv_rotary_t *rotary, int64_t num_tokens,
                               void *stream) {
  WKV_CHECK_ARG(norm != nullptr, "norm must be given (wkv_rotary_axes turns heads without one)");
  return norm_rotary_call(dtype, q, q_stride_t, q_stride_h, q_out, qo_stride_t, qo_stride_h, num_q_heads, k, k_stride_t,
                          k_stride_h, k_out, ko_stride_t, ko_stride_h, num_k_heads, head_dim, norm, rotary, num_tokens,
                          stream);
}

extern "C" int wkv_turn_heads(int32_t dtype, const void *q, int64_t q_stride_t, int64_t q_stride_h, void *q_out,
                              int64_t qo_stride_t, int64_t qo_stride_h, int32_t num_q_heads, const void *k,
                              int64_t k_stride_t, int64_t k_stride_h, void *k_out, int64_t ko_stride_t,
                              int64_t ko_stride_h, int32_t num_k_heads, int32_t head_dim, const wkv_rotary_t *rotary,
                              int64_t num_tokens, void *stream) {
  WKV_CHECK_ARG(rotary != nullptr, "rotary must be given");
  return norm_rotary_call(dtype, q, q_stride_t, q_stride_h, q_out, qo_stride_t, qo_stride_h, num_q_heads, k, k_stride_t,
                          k_stride_h, k_out, ko_stride_t, ko_stride_h, num_k_heads, head_dim, nullptr, rotary,
                          num_tokens, stream);
}

namespace {

// Most workgroups of the backward launch: the three waves a SIMD that its registers allow (8,191 tokens of 24
// heads of 128, bf16: 36 us; 512 or 1,024 workgroups 46).
constexpr int64_t kGradWorkgroups = 768;

// The most rows of sums that a kind's workgroups leave: one each, of their share of the workgroups, or, where
// each head has sums of its own, one a head from every workgroup along the tokens, of which a range of heads (a
// wave's: 1,024 elements at most) has its share.
struct GradSums {
  int64_t rows = 0;
  GradSums(int64_t tokens, int heads, int all_heads, int D, bool each) {
    if (tokens == 0 || heads == 0) return;
    const int64_t ranges = (static_cast<int64_t>(heads) * D + 1023) / 1024;
    rows = each ? std::min(share(kGradWorkgroups, ranges), most(tokens)) * heads
                : std::min(share(kGradWorkgroups * heads, all_heads), most(tokens) * (long_row(heads, D) ? heads : 1));
  }
  static int64_t share(int64_t of, int64_t among) { return std::max<int64_t>(of / among, 1); }
  static bool long_row(int heads, int D) { return heads * D >= 4096; }  // (taken by ranges also with one weight)
  static int64_t most(int64_t tokens) { return (tokens + kNormWaves - 1) / kNormWaves; }
};

}  // namespace

extern "C" int64_t wkv_norm_rotary_workspace_size(int64_t num_tokens, int32_t num_q_heads, int32_t num_k_heads,
                                                  int32_t head_dim, int32_t q_weight_each_head,
                                                  int32_t k_weight_each_head) {
  if (num_tokens < 0 || num_tokens > INT32_MAX || num_q_heads < 0 || num_k_heads < 0 || num_q_heads > 65535 ||
      num_k_heads > 65535 || head_dim <= 0 || head_dim > WKV_ROTARY_MAX_DIM)
    return -1;
  const int all = num_q_heads + num_k_heads;
  return (GradSums(num_tokens, num_q_heads, all, head_dim, q_weight_each_head != 0).rows +
          GradSums(num_tokens, num_k_heads, all, head_dim, k_weight_each_head != 0).rows) *
         head_dim * static_cast<int64_t>(sizeof(float));
}

extern "C" int wkv_norm_rotary_backward(int32_t dtype, const void *q, int64_t q_stride_t, int64_t q_stride_h,
                                        const void *q_grad, int64_t qg_stride_t, int64_t qg_stride_h, void *dq,
                                        int64_t dq_stride_t, int64_t dq_stride_h, int32_t num_q_heads, const void *k,
                                        int64_t k_stride_t, int64_t k_stride_h, const void *k_grad,
                                        int64_t kg_stride_t, int64_t kg_stride_h, void *dk, int64_t dk_stride_t,
                                        int64_t dk_stride_h, int32_t num_k_heads, int32_t head_dim,
                                        const wkv_head_norm_t *norm, const wkv_rotary_t *rotary, void *dq_weight,
                                        void *dk_weight, int64_t num_tokens, void *workspace, int64_t workspace_bytes,
                                        void *stream) {
  WKV_CHECK_ARG(norm != nullptr, "norm must be given");
  if (const int rc = check_norm_call(dtype, num_q_heads, num_k_heads, head_dim, norm, rotary, num_tokens)) return rc;
  const int esz = dtype == 0 ? 4 : 2, wsz = norm->weight_dtype == 0 ? 4 : 2;
  if (num_q_heads + num_k_heads == 0) return WKV_OK;
  auto kind_ok = [&](int heads, const void *x, int64_t xt, int64_t xh, const void *g, int64_t gt, int64_t gh,
                     const void *d, int64_t dt, int64_t dh) {
    return heads == 0 || num_tokens == 0 ||
           (rows_ok(x, xt, xh, esz) && rows_ok(g, gt, gh, esz) && (d == nullptr || rows_ok(d, dt, dh, esz)));
  };
  WKV_CHECK_ARG(kind_ok(num_q_heads, q, q_stride_t, q_stride_h, q_grad, qg_stride_t, qg_stride_h, dq, dq_stride_t, dq_stride_h) &&
                    kind_ok(num_k_heads, k, k_stride_t, k_stride_h, k_grad, kg_stride_t, kg_stride_h, dk, dk_stride_t, dk_stride_h),
                "q / k and their gradients must be non-NULL, aligned to their elements, their strides non-negative");
  WKV_CHECK_ARG((dq_weight == nullptr || (num_q_heads > 0 && norm->q_weight != nullptr)) &&
                    (dk_weight == nullptr || (num_k_heads > 0 && norm->k_weight != nullptr)),
                "a gradient of a weight that is not there");
  const bool dw = dq_weight != nullptr || dk_weight != nullptr;
  const int half = rotary != nullptr ? rotary->rotary_dim / 2 : 0;
  const bool inter = rotary != nullptr && rotary->interleaved != 0;
  const bool q_each = norm->q_weight != nullptr && norm->q_weight_stride_h != 0;
  const bool k_each = norm->k_weight != nullptr && norm->k_weight_stride_h != 0;
  const int H = num_q_heads + num_k_heads;
  const GradSums sq(num_tokens, num_q_heads, H, head_dim, q_each), sk(num_tokens, num_k_heads, H, head_dim, k_each);
  const int64_t need = (sq.rows + sk.rows) * head_dim * static_cast<int64_t>(sizeof(float));
  WeightGrads sum{static_cast<const float *>(workspace), dq_weight, dk_weight, q_each ? num_q_heads : num_q_heads > 0,
                  k_each ? num_k_heads : num_k_heads > 0, 0, 0, head_dim, norm->weight_dtype};
  if (dw)
    WKV_CHECK_ARG(need == 0 || (workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= need),
                  "workspace must hold wkv_norm_rotary_workspace_size() bytes, 16-byte aligned");
  auto s = static_cast<hipStream_t>(stream);
  if (num_tokens > 0) {
    NormGradArgs a{};
    const GradRows rq{q, q_grad, dq, q_stride_t, q_stride_h, qg_stride_t, qg_stride_h, dq_stride_t, dq_stride_h};
    const GradRows rk{k, k_grad, dk, k_stride_t, k_stride_h, kg_stride_t, kg_stride_h, dk_stride_t, dk_stride_h};
    a.n = head_norm(norm);
    a.a = angles(rotary);
    a.a.sign = -a.a.sign;
    a.tokens = num_tokens;
    a.partial = dw ? static_cast<float *>(workspace) : nullptr;
    Widths w(esz, head_dim, half, inter);
    auto fit = [&](int heads, const GradRows &r, const void *weight, int64_t ws) {
      if (heads == 0) return;
      w.rows(r.x, r.xt, r.xh);
      w.rows(r.g, r.gt, r.gh);
      if (r.dx != nullptr) w.rows(r.dx, r.dt, r.dh);
      w.weights(weight, ws, wsz);
    };
    fit(num_q_heads, rq, norm->q_weight, norm->q_weight_stride_h);
    fit(num_k_heads, rk, norm->k_weight, norm->k_weight_stride_h);
    a.r = row_units(head_dim, half, w.v);
    const int groups = 64 >> a.r.log_lanes;
    // Long rows of heads go by ranges with one weight too (16,384 tokens of 40 heads of 128, bf16: 98 us, 106 where a
    // wave walks a token's heads; fp32 169 and 195), but not short ones (8,191 of 24: 40 and 37.5) or where a token's
    // angles, which each range forms, cost more (32 of 256: 92 and 83). The workgroups are dealt by what a
    // token of a kind costs, in heads: a range costs a whole wave.
    auto in_ranges = [&](int heads, bool each, const GradSums &most) {
      return each || (GradSums::long_row(heads, head_dim) && half <= 64 && most.rows >= (heads + groups - 1) / groups);
    };
    const bool q_split = in_ranges(num_q_heads, q_each, sq), k_split = in_ranges(num_k_heads, k_each, sk);
    auto ranges = [&](int heads, bool split) { return heads == 0 ? 0 : split ? (heads + groups - 1) / groups : 1; };
    const int64_t cost_q = q_split ? ranges(num_q_heads, true) * groups : num_q_heads;
    const int64_t cost_k = k_split ? ranges(num_k_heads, true) * groups : num_k_heads;
    auto kind = [&](const GradRows &r, const void *weight, int64_t ws, int heads, bool each, bool split, int64_t cost,
                    const GradSums &most, int64_t first) {
      GradKind k{r, weight, ws, heads, each, split, ranges(heads, split), 0, 0, first};
      if (heads == 0) return k;
      const int64_t wgs = std::min(GradSums::share(kGradWorkgroups * cost, (cost_q + cost_k) * k.ranges), GradSums::most(num_tokens));
      k.wgs = static_cast<int>(std::min(wgs, most.rows / (each ? heads : k.ranges)));  // (what the workspace is for)
      // Two tokens a block in ranges (16,384 tokens of 40 heads of 128, bf16: 98 us, 104 of one, 105 of four);
      // else as many as give every group of lanes a head (8,192 of 16 + 16 heads of 256: one 83, two 99).
      const int64_t waves = static_cast<int64_t>(k.wgs) * kNormWaves;
      while (split ? k.log_tg < 1 && (num_tokens >> 1) >= waves
                   : (heads << k.log_tg) <= groups && (2 << k.log_tg) <= groups && (num_tokens >> (k.log_tg + 1)) >= waves)
        ++k.log_tg;
      return k;
    };
    a.q = kind(rq, norm->q_weight, norm->q_weight_stride_h, num_q_heads, q_each, q_split, cost_q, sq, 0);
    sum.q_wgs = a.q.wgs * (q_each ? 1 : a.q.ranges);
    a.k = kind(rk, norm->k_weight, norm->k_weight_stride_h, num_k_heads, k_each, k_split, cost_k, sk,
               static_cast<int64_t>(sum.q_wgs) * sum.q_rows);
    sum.k_wgs = a.k.wgs * (k_each ? 1 : a.k.ranges);
    const int64_t grid = static_cast<int64_t>(a.q.ranges) * a.q.wgs + static_cast<int64_t>(a.k.ranges) * a.k.wgs;
    WKV_CHECK_ARG(grid <= kMaxWorkgroups, "too many tokens and heads for one launch");
    const bool far = num_tokens * H * head_dim * esz >= (64 << 20);
    const int log_tg = a.q.log_tg > a.k.log_tg ? a.q.log_tg : a.k.log_tg;
    const size_t turns = (static_cast<size_t>(kNormWaves) << log_tg) * half * sizeof(float2);
    const size_t sums = static_cast<size_t>(kNormWaves) * (q_each || k_each ? groups : 1) * head_dim * sizeof(float);
    const size_t lds = turns > sums ? turns : sums;
    with_types(dtype, w.v, inter, [&](auto zero, auto v, auto in) {
      using T = decltype(zero);
      if (dw) launch_norm_grad<T, decltype(v)::value, decltype(in)::value, true>(a, far, static_cast<unsigned>(grid), lds, s);
      else launch_norm_grad<T, decltype(v)::value, decltype(in)::value, false>(a, far, static_cast<unsigned>(grid), lds, s);
    });
    WKV_CHECK_LAUNCH("norm_rotary_backward");
  }
  if (dw) {
    const dim3 grid(static_cast<unsigned>(sum.q_rows + sum.k_rows), static_cast<unsigned>((head_dim + 63) / 64));
    norm_weight_grad_kernel<<<grid, 64 * kSumWaves, 0, s>>>(sum);
    WKV_CHECK_LAUNCH("norm_weight_grad");
  }
  return WKV_OK;
}
