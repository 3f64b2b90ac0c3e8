// Norms of queries and keys for each head with the rotary positions in the same
// pass, forward and backward (gfx950). The mathematics: norm_rotary_dev.h.
//
// Forward: a workgroup takes a tile of tokens and some or all of their heads. It
// forms the tile's angles once, in LDS, and walks the tile's rows, a few in flight
// for each group of lanes.
//
// Backward, from the inputs and the outputs' gradient g: with z = R^T g, m = z (w + offset), r the
// reciprocal root mean square,
//   dx = r (m - x r^2 mean(m x)),   dw = sum over rows of z x r.
// A group of lanes keeps its elements of dw in registers over all the rows that
// it takes; workgroups leave their sums in the workspace, and a second kernel
// adds them up, in an order that the sizes alone give.
#include <type_traits>

#include "norm_rotary_dev.h"

namespace wkv {

constexpr int kNormThreads = 256;

struct NormRotaryArgs {
  HeadRows q, k;
  HeadNorm n;
  Angles a;
  RowUnits r;
  int64_t tokens;
  int Hq, H;  // query heads; query and key heads
  int tile;   // tokens of a workgroup
  FastDiv per, last;  // heads of a workgroup; of the last along the grid's y
};

template <class T, int V, bool INTER, int U, bool FAR>
__global__ __launch_bounds__(kNormThreads) void norm_rotary_kernel(NormRotaryArgs a) {
  typedef typename VecOf<T, V>::type Vec;
  extern __shared__ float2 turn[];
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * a.tile;
  const int nt = a.tokens - t0 < a.tile ? static_cast<int>(a.tokens - t0) : a.tile;
  const FastDiv heads = blockIdx.y + 1 == gridDim.y ? a.last : a.per;
  tile_angles(a.a, t0, nt, kNormThreads, turn);
  __syncthreads();
  norm_turn_rows<T, V, INTER, U, U == 1 ? 2 : 1, FAR>(
      a.r, a.n, a.Hq, turn, nt, heads, blockIdx.y * a.per.d, kNormThreads,
      [&](int t, int h) {
        const HeadRows &s = h < a.Hq ? a.q : a.k;
        return static_cast<const T *>(s.x) + (t0 + t) * s.xt + (h < a.Hq ? h : h - a.Hq) * s.xh;
      },
      [&](int t, int h, int e, Vec v) {
        const HeadRows &s = h < a.Hq ? a.q : a.k;
        Vec *y = reinterpret_cast<Vec *>(static_cast<T *>(s.y) + (t0 + t) * s.yt + (h < a.Hq ? h : h - a.Hq) * s.yh + e);
        if (FAR)
          __builtin_nontemporal_store(v, y);
        else
          *y = v;
      });
}

// ---------------------------------------------------------------------------
// Backward.
struct GradRows {
  const void *x, *g;
  void *dx;  // nullptr: not asked for
  int64_t xt, xh, gt, gh, dt, dh;
};

// A workgroup's share: `heads` heads of one kind from one on, every gridth tile.
struct NormGradArgs {
  GradRows q, k;
  HeadNorm n;
  Angles a;  // sign: the transpose's
  RowUnits r;
  int64_t tokens, tiles;
  int tile;
  int q_ranges, k_ranges;  // ranges of heads: one of all, or each head's own
  int q_wgs, k_wgs;        // workgroups of a range
  FastDiv q_per, k_per;    // heads of a range
  float *partial;          // [ranges' workgroups, D]; nullptr: no weight's gradient
};

template <class T, int V, bool INTER, int U, bool FAR, bool DW>
__global__ __launch_bounds__(kNormThreads) void norm_rotary_grad_kernel(NormGradArgs a) {
  typedef typename VecOf<T, V>::type Vec;
  extern __shared__ float2 turn[];
  const int nq = a.q_ranges * a.q_wgs;
  const bool is_q = static_cast<int>(blockIdx.x) < nq;
  const int b = is_q ? blockIdx.x : blockIdx.x - nq;
  const int wgs = is_q ? a.q_wgs : a.k_wgs;
  const FastDiv heads = is_q ? a.q_per : a.k_per;
  const int range = b / wgs, h0 = range * heads.d;
  const GradRows s = is_q ? a.q : a.k;
  const void *w = is_q ? a.n.qw : a.n.kw;
  const int64_t ws = is_q ? a.n.qws : a.n.kws;
  const int lanes = 1 << a.r.log_lanes, group = threadIdx.x >> a.r.log_lanes, u0 = threadIdx.x & (lanes - 1);
  const int groups = kNormThreads >> a.r.log_lanes;
  const float inv_d = 1.f / static_cast<float>(a.r.D);
  float acc0[U][V], acc1[U][V];
#pragma unroll
  for (int j = 0; j < U; ++j)
#pragma unroll
    for (int v = 0; v < V; ++v) acc0[j][v] = acc1[j][v] = 0.f;
  constexpr int N = U == 1 ? 2 : 1;
  for (int64_t tile = b - range * wgs; tile < a.tiles; tile += wgs) {  // uniform
    const int64_t t0 = tile * a.tile;
    const int nt = a.tokens - t0 < a.tile ? static_cast<int>(a.tokens - t0) : a.tile;
    __syncthreads();
    tile_angles(a.a, t0, nt, kNormThreads, turn);
    __syncthreads();
    const int rows = nt * heads.d;
    for (int r0 = 0; r0 < rows; r0 += groups * N) {
      Vec x0[N][U], x1[N][U], g0[N][U], g1[N][U];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int r = r0 + groups * k + group;
        const int t = r / heads, h = h0 + r - t * heads.d;
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const int u = u0 + lanes * j;
          if (r < rows && u < a.r.units) {
            int e0, e1;
            unit_runs<V, INTER>(a.r, u, e0, e1);
            const T *x = static_cast<const T *>(s.x) + (t0 + t) * s.xt + h * s.xh;
            const T *g = static_cast<const T *>(s.g) + (t0 + t) * s.gt + h * s.gh;
            const Vec *px0 = reinterpret_cast<const Vec *>(x + e0), *px1 = reinterpret_cast<const Vec *>(x + e1);
            const Vec *pg0 = reinterpret_cast<const Vec *>(g + e0), *pg1 = reinterpret_cast<const Vec *>(g + e1);
            x0[k][j] = FAR ? __builtin_nontemporal_load(px0) : *px0;
            x1[k][j] = FAR ? __builtin_nontemporal_load(px1) : *px1;
            g0[k][j] = FAR ? __builtin_nontemporal_load(pg0) : *pg0;
            g1[k][j] = FAR ? __builtin_nontemporal_load(pg1) : *pg1;
          } else {
            x0[k][j] = x1[k][j] = g0[k][j] = g1[k][j] = Vec{};
          }
        }
      }
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int r = r0 + groups * k + group;
        const int t = r / heads, h = h0 + r - t * heads.d;
        float f0[U][V], f1[U][V], z0[U][V], z1[U][V], m0[U][V], m1[U][V], ss = 0.f, sm = 0.f;
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const int u = u0 + lanes * j;
          int e0 = 0, e1 = 0;
          if (r < rows && u < a.r.units) unit_runs<V, INTER>(a.r, u, e0, e1);
          widen<V, T>(x0[k][j], f0[j]);
          widen<V, T>(x1[k][j], f1[j]);
          widen<V, T>(g0[k][j], z0[j]);
          widen<V, T>(g1[k][j], z1[j]);
          // (a lane without a unit holds zeros, and turns them by some token's angles)
          turn_unit<V, INTER>(turn + (r < rows ? t * a.a.half.d : 0), a.r.half, e0, e1, z0[j], z1[j]);
          float w0[V], w1[V];
          const int64_t wh = r < rows ? h * ws : 0;
          load_weights<T, V>(a.n, w, wh + e0, w0);
          load_weights<T, V>(a.n, w, wh + e1, w1);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            m0[j][v] = z0[j][v] * w0[v];
            m1[j][v] = z1[j][v] * w1[v];
            ss = __builtin_fmaf(f0[j][v], f0[j][v], __builtin_fmaf(f1[j][v], f1[j][v], ss));
            sm = __builtin_fmaf(m0[j][v], f0[j][v], __builtin_fmaf(m1[j][v], f1[j][v], sm));
          }
        }
        ss = group_sum(ss, a.r.log_lanes);
        sm = group_sum(sm, a.r.log_lanes);
        const float inv = rsqrtf(__builtin_fmaf(ss, inv_d, a.n.eps));
        const float back = sm * inv_d * inv * inv;
        if (DW) {
#pragma unroll
          for (int j = 0; j < U; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) {
              acc0[j][v] = __builtin_fmaf(z0[j][v], f0[j][v] * inv, acc0[j][v]);
              acc1[j][v] = __builtin_fmaf(z1[j][v], f1[j][v] * inv, acc1[j][v]);
            }
        }
        if (r >= rows || s.dx == nullptr) continue;
        T *y = static_cast<T *>(s.dx) + (t0 + t) * s.dt + h * s.dh;
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const int u = u0 + lanes * j;
          if (u >= a.r.units) continue;
          int e0, e1;
          unit_runs<V, INTER>(a.r, u, e0, e1);
          Vec o0, o1;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            o0[v] = static_cast<T>(inv * __builtin_fmaf(-back, f0[j][v], m0[j][v]));
            o1[v] = static_cast<T>(inv * __builtin_fmaf(-back, f1[j][v], m1[j][v]));
          }
          Vec *p0 = reinterpret_cast<Vec *>(y + e0), *p1 = reinterpret_cast<Vec *>(y + e1);
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
  }
  if (!DW) return;
  // The groups' sums: of a wave's groups by butterflies, of the waves through LDS.
  float *sums = reinterpret_cast<float *>(turn);  // [waves, D]
  __syncthreads();
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int j = 0; j < U; ++j) {
    const int u = u0 + lanes * j;
    int e0 = 0, e1 = 0;
    if (u < a.r.units) unit_runs<V, INTER>(a.r, u, e0, e1);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float s0 = acc0[j][v], s1 = acc1[j][v];
      for (int o = lanes; o < 64; o *= 2) {  // uniform
        s0 += __shfl_xor(s0, o, 64);
        s1 += __shfl_xor(s1, o, 64);
      }
      if (u < a.r.units && (threadIdx.x & 63) < lanes) {
        sums[wave * a.r.D + e0 + v] = s0;
        sums[wave * a.r.D + e1 + v] = s1;
      }
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < a.r.D; d += kNormThreads) {
    float s0 = 0.f;
#pragma unroll
    for (int i = 0; i < kNormThreads / 64; ++i) s0 += sums[i * a.r.D + d];
    a.partial[static_cast<int64_t>(blockIdx.x) * a.r.D + d] = s0;
  }
}

// The weights' gradients from the workgroups' sums: a workgroup adds up 64
// elements of one range, a sixteenth of the sums each wave.
constexpr int kSumWaves = 16;
struct WeightGrads {
  const float *partial;
  void *dq, *dk;  // nullptr: not asked for
  int q_ranges, q_wgs, k_wgs, D;
  int dtype;  // of the gradients: 0 fp32, 1 bf16, 2 fp16
};

__global__ __launch_bounds__(64 * kSumWaves) void norm_weight_grad_kernel(WeightGrads a) {
  __shared__ float sums[kSumWaves][64];
  const bool is_q = static_cast<int>(blockIdx.x) < a.q_ranges;
  const int range = is_q ? blockIdx.x : blockIdx.x - a.q_ranges;
  void *out = is_q ? a.dq : a.dk;
  if (out == nullptr) return;  // uniform
  const int n = is_q ? a.q_wgs : a.k_wgs;
  const int64_t first = is_q ? static_cast<int64_t>(range) * n : static_cast<int64_t>(a.q_ranges) * a.q_wgs + static_cast<int64_t>(range) * n;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, d = blockIdx.y * 64 + lane;
  float s = 0.f;
  if (d < a.D) {
#pragma unroll 8
    for (int i = wave; i < n; i += kSumWaves) s += a.partial[(first + i) * a.D + d];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || d >= a.D) return;
#pragma unroll
  for (int i = 1; i < kSumWaves; ++i) s += sums[i][lane];
  const int64_t at = static_cast<int64_t>(range) * a.D + d;
  if (a.dtype == 0)
    static_cast<float *>(out)[at] = s;
  else if (a.dtype == 1)
    static_cast<__bf16 *>(out)[at] = static_cast<__bf16>(s);
  else
    static_cast<_Float16 *>(out)[at] = static_cast<_Float16>(s);
}

// ---------------------------------------------------------------------------
// Host.
// The forward launch.
template <class T, int V, bool INTER>
static void launch_norm(const NormRotaryArgs &a, bool far, dim3 grid, size_t lds, hipStream_t s) {
  constexpr bool WIDE = V * sizeof(T) == 16;
  if (a.r.units > 64) {
    if constexpr (V <= 2) norm_rotary_kernel<T, V, INTER, 4, false><<<grid, kNormThreads, lds, s>>>(a);
    return;
  }
  if constexpr (WIDE) {
    if (far) {
      norm_rotary_kernel<T, V, INTER, 1, true><<<grid, kNormThreads, lds, s>>>(a);
      return;
    }
  }
  norm_rotary_kernel<T, V, INTER, 1, false><<<grid, kNormThreads, lds, s>>>(a);
}

template <class T, int V, bool INTER>
static void launch_norm_grad(const NormGradArgs &a, bool far, unsigned grid, size_t lds, hipStream_t s) {
  constexpr bool WIDE = V * sizeof(T) == 16;
  const bool dw = a.partial != nullptr;
  if (a.r.units > 64) {
    if constexpr (V <= 2) {
      if (dw) norm_rotary_grad_kernel<T, V, INTER, 4, false, true><<<grid, kNormThreads, lds, s>>>(a);
      else norm_rotary_grad_kernel<T, V, INTER, 4, false, false><<<grid, kNormThreads, lds, s>>>(a);
    }
    return;
  }
  if constexpr (WIDE) {
    if (far) {
      if (dw) norm_rotary_grad_kernel<T, V, INTER, 1, true, true><<<grid, kNormThreads, lds, s>>>(a);
      else norm_rotary_grad_kernel<T, V, INTER, 1, true, false><<<grid, kNormThreads, lds, s>>>(a);
      return;
    }
  }
  if (dw) norm_rotary_grad_kernel<T, V, INTER, 1, false, true><<<grid, kNormThreads, lds, s>>>(a);
  else norm_rotary_grad_kernel<T, V, INTER, 1, false, false><<<grid, kNormThreads, lds, s>>>(a);
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

// Tokens whose angles take 8 KB.
int tile_tokens(int half) {
  const int t = half > 0 ? 1024 / half : 16;
  return t < 1 ? 1 : t > 16 ? 16 : t;
}

}  // namespace

extern "C" int wkv_norm_rotary(int32_t dtype, const void *q, int64_t q_stride_t, int64_t q_stride_h, void *q_out,
                               int64_t qo_stride_t, int64_t qo_stride_h, int32_t num_q_heads, const void *k,
                               int64_t k_stride_t, int64_t k_stride_h, void *k_out, int64_t ko_stride_t,
                               int64_t ko_stride_h, int32_t num_k_heads, int32_t head_dim,
                               const wkv_head_norm_t *norm, const wkv_rotary_t *rotary, int64_t num_tokens,
                               void *stream) {
  WKV_CHECK_ARG(norm != nullptr, "norm must be given (wkv_rotary_axes turns heads without one)");
  if (const int rc = check_norm_call(dtype, num_q_heads, num_k_heads, head_dim, norm, rotary, num_tokens)) return rc;
  const int H = num_q_heads + num_k_heads, esz = dtype == 0 ? 4 : 2;
  if (num_tokens == 0 || H == 0) return WKV_OK;
  WKV_CHECK_ARG((num_q_heads == 0 || (rows_ok(q, q_stride_t, q_stride_h, esz) && rows_ok(q_out, qo_stride_t, qo_stride_h, esz))) &&
                    (num_k_heads == 0 || (rows_ok(k, k_stride_t, k_stride_h, esz) && rows_ok(k_out, ko_stride_t, ko_stride_h, esz))),
                "q / k and their outputs must be non-NULL, aligned to their elements, their strides non-negative");
  const int half = rotary != nullptr ? rotary->rotary_dim / 2 : 0;
  const bool inter = rotary != nullptr && rotary->interleaved != 0;
  NormRotaryArgs a{};
  a.q = HeadRows{q, q_out, q_stride_t, q_stride_h, qo_stride_t, qo_stride_h};
  a.k = HeadRows{k, k_out, k_stride_t, k_stride_h, ko_stride_t, ko_stride_h};
  a.n = head_norm(norm);
  a.a = angles(rotary);
  a.tokens = num_tokens;
  a.Hq = num_q_heads;
  a.H = H;
  Widths w(esz, head_dim, half, inter);
  const int wsz = norm->weight_dtype == 0 ? 4 : 2;
  if (num_q_heads > 0) {
    w.rows(q, q_stride_t, q_stride_h);
    w.rows(q_out, qo_stride_t, qo_stride_h);
    w.weights(norm->q_weight, norm->q_weight_stride_h, wsz);
  }
  if (num_k_heads > 0) {
    w.rows(k, k_stride_t, k_stride_h);
    w.rows(k_out, ko_stride_t, ko_stride_h);
    w.weights(norm->k_weight, norm->k_weight_stride_h, wsz);
  }
  a.r = row_units(head_dim, half, w.v);
  // With too few tokens for the chip, smaller tiles, then their heads over more workgroups.
  a.tile = tile_tokens(half);
  while (a.tile > 1 && (num_tokens + a.tile - 1) / a.tile < 1024) a.tile /= 2;
  const int64_t tiles = (num_tokens + a.tile - 1) / a.tile;
  const int groups = kNormThreads >> a.r.log_lanes;
  const int64_t want = (1024 + tiles - 1) / tiles, most = (H + groups - 1) / groups;
  const int split = static_cast<int>(want < most ? want : most);
  a.per = fast_div((H + split - 1) / split);
  const int ny = (H + a.per.d - 1) / a.per.d;
  a.last = fast_div(H - (ny - 1) * a.per.d);
  const bool far = num_tokens * H * head_dim * esz >= (64 << 20);
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(ny));
  const size_t lds = static_cast<size_t>(a.tile) * half * sizeof(float2);
  auto s = static_cast<hipStream_t>(stream);
  with_types(dtype, w.v, inter, [&](auto zero, auto v, auto in) {
    launch_norm<decltype(zero), decltype(v)::value, decltype(in)::value>(a, far, grid, lds, s);
  });
  WKV_CHECK_LAUNCH("norm_rotary");
  return WKV_OK;
}

namespace {

// Workgroups of the backward launch along the tokens, for each kind of heads.
struct GradGrid {
  int tile, q_ranges, k_ranges, q_wgs, k_wgs;
  int64_t tiles;
  GradGrid(int64_t tokens, int Hq, int Hk, int half, bool q_each, bool k_each) {
    tile = tile_tokens(half);
    while (tile > 1 && (tokens + tile - 1) / tile < 512) tile /= 2;
    tiles = (tokens + tile - 1) / tile;
    q_ranges = Hq == 0 ? 0 : q_each ? Hq : 1;
    k_ranges = Hk == 0 ? 0 : k_each ? Hk : 1;
    const int64_t total = 1024, H = Hq + Hk > 0 ? Hq + Hk : 1;
    auto wgs = [&](int heads, int ranges) -> int {
      if (ranges == 0) return 0;
      int64_t n = (total * heads + H * ranges - 1) / (H * ranges);
      n = n < 1 ? 1 : n;
      return static_cast<int>(n < tiles ? n : tiles);
    };
    q_wgs = wgs(Hq, q_ranges);
    k_wgs = wgs(Hk, k_ranges);
  }
  int64_t count() const { return static_cast<int64_t>(q_ranges) * q_wgs + static_cast<int64_t>(k_ranges) * k_wgs; }
};

}  // namespace

extern "C" int64_t wkv_norm_rotary_workspace_size(int64_t num_tokens, int32_t num_q_heads, int32_t num_k_heads,
                                                  int32_t head_dim, int32_t rotary_dim, int32_t q_weight_each_head,
                                                  int32_t k_weight_each_head) {
  if (num_tokens < 0 || num_tokens > INT32_MAX || num_q_heads < 0 || num_k_heads < 0 || num_q_heads > 65535 ||
      num_k_heads > 65535 || head_dim <= 0 || head_dim > WKV_ROTARY_MAX_DIM || rotary_dim < 0 || rotary_dim > head_dim)
    return -1;
  const GradGrid g(num_tokens, num_q_heads, num_k_heads, rotary_dim / 2, q_weight_each_head != 0, k_weight_each_head != 0);
  return g.count() * head_dim * static_cast<int64_t>(sizeof(float));
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
  const GradGrid g(num_tokens, num_q_heads, num_k_heads, half, dq_weight != nullptr && norm->q_weight_stride_h != 0,
                   dk_weight != nullptr && norm->k_weight_stride_h != 0);
  if (dw)
    WKV_CHECK_ARG(g.count() == 0 || (workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 &&
                      workspace_bytes >= g.count() * head_dim * static_cast<int64_t>(sizeof(float))),
                  "workspace must hold wkv_norm_rotary_workspace_size() bytes, 16-byte aligned");
  auto s = static_cast<hipStream_t>(stream);
  if (num_tokens > 0) {
    NormGradArgs a{};
    a.q = GradRows{q, q_grad, dq, q_stride_t, q_stride_h, qg_stride_t, qg_stride_h, dq_stride_t, dq_stride_h};
    a.k = GradRows{k, k_grad, dk, k_stride_t, k_stride_h, kg_stride_t, kg_stride_h, dk_stride_t, dk_stride_h};
    a.n = head_norm(norm);
    a.a = angles(rotary);
    a.a.sign = -a.a.sign;
    a.tokens = num_tokens;
    a.tiles = g.tiles;
    a.tile = g.tile;
    a.q_ranges = g.q_ranges;
    a.k_ranges = g.k_ranges;
    a.q_wgs = g.q_wgs;
    a.k_wgs = g.k_wgs;
    a.q_per = fast_div(g.q_ranges > 0 ? num_q_heads / g.q_ranges : 1);
    a.k_per = fast_div(g.k_ranges > 0 ? num_k_heads / g.k_ranges : 1);
    a.partial = dw ? static_cast<float *>(workspace) : nullptr;
    Widths w(esz, head_dim, half, inter);
    auto kind = [&](int heads, const GradRows &r, const void *weight, int64_t ws) {
      if (heads == 0) return;
      w.rows(r.x, r.xt, r.xh);
      w.rows(r.g, r.gt, r.gh);
      if (r.dx != nullptr) w.rows(r.dx, r.dt, r.dh);
      w.weights(weight, ws, wsz);
    };
    kind(num_q_heads, a.q, norm->q_weight, norm->q_weight_stride_h);
    kind(num_k_heads, a.k, norm->k_weight, norm->k_weight_stride_h);
    a.r = row_units(head_dim, half, w.v);
    const bool far = num_tokens * (num_q_heads + num_k_heads) * head_dim * esz >= (64 << 20);
    const size_t turns = static_cast<size_t>(g.tile) * half * sizeof(float2);
    const size_t sums = static_cast<size_t>(kNormThreads / 64) * head_dim * sizeof(float);
    const size_t lds = turns > sums ? turns : sums;
    with_types(dtype, w.v, inter, [&](auto zero, auto v, auto in) {
      launch_norm_grad<decltype(zero), decltype(v)::value, decltype(in)::value>(
          a, far, static_cast<unsigned>(g.count()), lds, s);
    });
    WKV_CHECK_LAUNCH("norm_rotary_backward");
  }
  if (dw) {
    WeightGrads a{static_cast<const float *>(workspace), dq_weight, dk_weight, g.q_ranges,
                  num_tokens > 0 ? g.q_wgs : 0, num_tokens > 0 ? g.k_wgs : 0, head_dim, norm->weight_dtype};
    const dim3 grid(static_cast<unsigned>(g.q_ranges + g.k_ranges), static_cast<unsigned>((head_dim + 63) / 64));
    norm_weight_grad_kernel<<<grid, 64 * kSumWaves, 0, s>>>(a);
    WKV_CHECK_LAUNCH("norm_weight_grad");
  }
  return WKV_OK;
}
