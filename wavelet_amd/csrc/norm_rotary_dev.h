// What the kernels that norm and turn heads share: a token's angles, and rows of
// heads taken by groups of lanes.
//
// A head x of D values is normed by its root mean square and turned,
//   n = x (mean(x^2) + eps)^-1/2 (w + offset),
//   y_a = s (n_a cos t - n_b sin t),  y_b = s (n_b cos t + n_a sin t)
// for its pairs (a, b), t = position * inv_freq[pair]; either step may be
// absent. All of it is float32 (angles float64, reduced in turns), rounded once.
//
// A row (one head of one token) belongs to a group of lanes, the power of two
// that holds its units, 64 at most: a unit is V pairs in two runs of V elements,
// (V u, V u + half) or with adjacent pairs (V u, V (u + units)), so that a lane
// moves 16 bytes at a time and both elements of a pair meet in one lane. The
// sum of squares is a butterfly over the group.
#pragma once

#include <cmath>

#include "wkv_common.h"

namespace wkv {

struct Angles {
  const int64_t *pos;  // rows of positions, one an axis
  int64_t axis_stride;
  const int32_t *axes;  // of every pair (nullptr: all of axis 0)
  int num_axes;
  const double *inv_freq;
  FastDiv half;  // turned pairs (0: none are)
  float scale, sign;
};

// Cosine and sine of pair i at token t, times the scale. A pair of an axis that is not there stays.
__device__ __forceinline__ float2 angle_at(const Angles &a, int64_t t, int i) {
  const int ax = a.axes != nullptr ? a.axes[i] : 0;
  double p = 0.;
  if (static_cast<unsigned>(ax) < static_cast<unsigned>(a.num_axes)) p = static_cast<double>(a.pos[ax * a.axis_stride + t]);
  const double x = p * a.inv_freq[i] * 0.15915494309189533577;  // 1 / 2 pi: the angle in turns
  float s, c;
  sincospif(2.f * static_cast<float>(x - rint(x)), &s, &c);
  return make_float2(c * a.scale, s * a.scale * a.sign);
}

struct HeadNorm {
  const void *qw, *kw;  // nullptr: ones
  int64_t qws, kws;     // between heads
  int on, wide;         // whether there is a norm; float32 weights
  float offset, eps;
};

// Rows of heads in and out; strides in elements: token, head.
struct HeadRows {
  const void *x;
  void *y;
  int64_t xt, xh, yt, yh;
};

// How a row's D values lie over its lanes.
struct RowUnits {
  int D, half;
  int units;   // of a row
  int turned;  // of them units that hold turned pairs only (pairs half apart)
  int log_lanes;
};

template <int V, bool INTER>
__device__ __forceinline__ void unit_runs(const RowUnits &a, int u, int &e0, int &e1) {
  if (INTER) {
    e0 = V > 1 ? V * u : 2 * u;
    e1 = V > 1 ? V * (u + a.units) : 2 * u + 1;
  } else if (u < a.turned) {
    e0 = V * u;
    e1 = e0 + a.half;
  } else {
    e0 = 2 * a.half + V * (u - a.turned);
    e1 = e0 + V * (a.units - a.turned);
  }
}

// The sum over a group of 2^log_lanes lanes, the same in each.
__device__ __forceinline__ float group_sum(float v, int log_lanes) {
  if (log_lanes > 0) v += lane_xor<1>(v);
  if (log_lanes > 1) v += lane_xor<2>(v);
  if (log_lanes > 2) v += lane_xor<4>(v);
  if (log_lanes > 3) v += lane_xor<8>(v);
  if (log_lanes > 4) v += lane_xor<16>(v);
  if (log_lanes > 5) v += lane_xor<32>(v);
  return v;
}

template <class T, int V>
struct VecOf {
  typedef __attribute__((__vector_size__(V * sizeof(T)))) T type;
};

template <int V, class T>
__device__ __forceinline__ void widen(const typename VecOf<T, V>::type &x, float *f) {
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = static_cast<float>(x[v]);
}

// V weights from element e on, the offset added.
template <class T, int V>
__device__ __forceinline__ void load_weights(const HeadNorm &n, const void *w, int64_t e, float *f) {
  if (w == nullptr) {
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = 1.f;
    return;
  }
  if (n.wide) {
    constexpr int W = V < 4 ? V : 4;
#pragma unroll
    for (int v = 0; v < V; v += W) {
      const auto x = *reinterpret_cast<const typename VecOf<float, W>::type *>(static_cast<const float *>(w) + e + v);
#pragma unroll
      for (int j = 0; j < W; ++j) f[v + j] = x[j] + n.offset;
    }
  } else {
    widen<V, T>(*reinterpret_cast<const typename VecOf<T, V>::type *>(static_cast<const T *>(w) + e), f);
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] += n.offset;
  }
}

// A pair turned by (cos, sin).
__device__ __forceinline__ void turn_pair(float2 cs, float &a, float &b) {
  const float x = a, y = b;
  a = __builtin_fmaf(x, cs.x, -(y * cs.y));
  b = __builtin_fmaf(y, cs.x, x * cs.y);
}

// A unit's pairs turned: runs fa from element e0 on and fb from e1 on, turn[]
// the angles of the row's token.
template <int V, bool INTER>
__device__ __forceinline__ void turn_unit(const float2 *turn, int half, int e0, int e1, float *fa, float *fb) {
  if (INTER && V > 1) {
#pragma unroll
    for (int v = 0; v < V; v += 2) {
      if ((e0 + v) / 2 < half) turn_pair(turn[(e0 + v) / 2], fa[v], fa[v + 1]);
      if ((e1 + v) / 2 < half) turn_pair(turn[(e1 + v) / 2], fb[v], fb[v + 1]);
    }
  } else {
    const int p = INTER ? e0 / 2 : e0;
    if (p < half) {
#pragma unroll
      for (int v = 0; v < V; ++v) turn_pair(turn[p + v], fa[v], fb[v]);
    }
  }
}

// A tile's angles, by the whole workgroup of `threads`; a barrier follows before they are read.
__device__ __forceinline__ void tile_angles(const Angles &a, int64_t t0, int nt, int threads, float2 *turn) {
  for (int i = threadIdx.x; i < nt * a.half.d; i += threads) {
    const int t = i / a.half;
    turn[i] = angle_at(a, t0 + t, i - t * a.half.d);
  }
}

// Rows of a tile of nt tokens, heads h0 .. h0 + heads.d - 1 of each, by a workgroup
// of `threads`: normed (if norm.on), turned by turn[], stored. N rows of a group of lanes in
// flight. src(t, h): where a row lies (nullptr: skipped); dst(t, h, e, v): stores its elements from e on.
template <class T, int V, bool INTER, int U, int N, bool FAR, class Src, class Dst>
__device__ __forceinline__ void norm_turn_rows(const RowUnits &ru, const HeadNorm &norm, int Hq, const float2 *turn,
                                               int nt, const FastDiv &heads, int h0, int threads, Src src, Dst dst) {
  typedef typename VecOf<T, V>::type Vec;
  const int lanes = 1 << ru.log_lanes, group = threadIdx.x >> ru.log_lanes, u0 = threadIdx.x & (lanes - 1);
  const int groups = threads >> ru.log_lanes, rows = nt * heads.d;
  const float inv_d = 1.f / static_cast<float>(ru.D);
  for (int r0 = 0; r0 < rows; r0 += groups * N) {
    Vec x0[N][U], x1[N][U];
    const T *x[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int r = r0 + groups * k + group;
      const int t = r / heads, h = h0 + r - t * heads.d;
      x[k] = r < rows ? src(t, h) : nullptr;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int u = u0 + lanes * j;
        if (x[k] != nullptr && u < ru.units) {
          int e0, e1;
          unit_runs<V, INTER>(ru, u, e0, e1);
          const Vec *p0 = reinterpret_cast<const Vec *>(x[k] + e0), *p1 = reinterpret_cast<const Vec *>(x[k] + e1);
          x0[k][j] = FAR ? __builtin_nontemporal_load(p0) : *p0;
          x1[k][j] = FAR ? __builtin_nontemporal_load(p1) : *p1;
        } else {
          x0[k][j] = Vec{};
          x1[k][j] = Vec{};
        }
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int r = r0 + groups * k + group;
      const int t = r / heads, h = h0 + r - t * heads.d;
      float f0[U][V], f1[U][V], ss = 0.f;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        widen<V, T>(x0[k][j], f0[j]);
        widen<V, T>(x1[k][j], f1[j]);
#pragma unroll
        for (int v = 0; v < V; ++v) ss = __builtin_fmaf(f0[j][v], f0[j][v], __builtin_fmaf(f1[j][v], f1[j][v], ss));
      }
      ss = group_sum(ss, ru.log_lanes);
      const float inv = norm.on ? rsqrtf(__builtin_fmaf(ss, inv_d, norm.eps)) : 1.f;
      if (x[k] == nullptr) continue;
      const void *w = h < Hq ? norm.qw : norm.kw;
      const int64_t wh = h < Hq ? h * norm.qws : (h - Hq) * norm.kws;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int u = u0 + lanes * j;
        if (u >= ru.units) continue;
        int e0, e1;
        unit_runs<V, INTER>(ru, u, e0, e1);
        float w0[V], w1[V];
        load_weights<T, V>(norm, w, wh + e0, w0);
        load_weights<T, V>(norm, w, wh + e1, w1);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          f0[j][v] *= inv * w0[v];
          f1[j][v] *= inv * w1[v];
        }
        turn_unit<V, INTER>(turn + t * ru.half, ru.half, e0, e1, f0[j], f1[j]);
        Vec o0, o1;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          o0[v] = static_cast<T>(f0[j][v]);
          o1[v] = static_cast<T>(f1[j][v]);
        }
        dst(t, h, e0, o0);
        dst(t, h, e1, o1);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host: the checks of a call's rotation and norm, and what the kernels take of them.
inline int check_rotary(const wkv_rotary_t *r, int head_dim, int64_t num_tokens) {
  WKV_CHECK_ARG(r->rotary_dim > 0 && r->rotary_dim % 2 == 0 && r->rotary_dim <= head_dim,
                "rotary_dim must be even and in [2, head_dim] (got %d)", r->rotary_dim);
  WKV_CHECK_ARG(std::isfinite(r->scale), "scale must be finite");
  WKV_CHECK_ARG(r->num_axes >= 1 && r->axis_stride >= 0, "num_axes must be positive, axis_stride non-negative");
  WKV_CHECK_ARG(r->reserved == 0, "rotary descriptor field `reserved` must be 0 (got %d)", r->reserved);
  WKV_CHECK_ARG(num_tokens == 0 || (r->positions != nullptr && reinterpret_cast<uintptr_t>(r->positions) % 8 == 0 &&
                    r->inv_freq != nullptr && reinterpret_cast<uintptr_t>(r->inv_freq) % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(r->axes) % 4 == 0),
                "positions and inv_freq must be non-NULL, int64 and float64, axes int32");
  return WKV_OK;
}

inline int check_norm_eps(float eps, float offset) {
  // (a square root of less than the smallest normal number would not be held)
  WKV_CHECK_ARG(std::isfinite(eps) && eps >= 1.17549435e-38f, "eps must be a positive normal number (got %g)", eps);
  WKV_CHECK_ARG(std::isfinite(offset), "weight_offset must be finite");
  return WKV_OK;
}

inline int check_head_norm(const wkv_head_norm_t *n, int dtype) {
  if (const int rc = check_norm_eps(n->eps, n->weight_offset)) return rc;
  WKV_CHECK_ARG(n->reserved == 0, "norm descriptor field `reserved` must be 0 (got %d)", n->reserved);
  if (n->q_weight == nullptr && n->k_weight == nullptr) return WKV_OK;
  WKV_CHECK_ARG(n->weight_dtype == 0 || n->weight_dtype == dtype, "weights must be fp32 or of the heads' type");
  const uintptr_t wsz = n->weight_dtype == 0 ? 4 : 2;
  WKV_CHECK_ARG(reinterpret_cast<uintptr_t>(n->q_weight) % wsz == 0 && reinterpret_cast<uintptr_t>(n->k_weight) % wsz == 0 &&
                    n->q_weight_stride_h >= 0 && n->k_weight_stride_h >= 0,
                "weights must be aligned to their elements, their strides non-negative");
  return WKV_OK;
}

inline HeadNorm head_norm(const wkv_head_norm_t *n) {
  if (n == nullptr) return HeadNorm{};
  return HeadNorm{n->q_weight, n->k_weight, n->q_weight_stride_h, n->k_weight_stride_h, 1, n->weight_dtype == 0,
                  n->weight_offset, n->eps};
}

inline Angles angles(const wkv_rotary_t *r) {
  if (r == nullptr) return Angles{nullptr, 0, nullptr, 0, nullptr, FastDiv{0u, 0}, 1.f, 1.f};
  return Angles{r->positions, r->axis_stride, r->axes, r->num_axes, r->inv_freq, fast_div(r->rotary_dim / 2), r->scale,
                r->inverse != 0 ? -1.f : 1.f};
}

inline RowUnits row_units(int D, int half, int v) {
  RowUnits r{D, half, D / (2 * v), half / v, 0};
  while (r.log_lanes < 6 && (1 << r.log_lanes) < r.units) ++r.log_lanes;
  return r;
}

// The elements of an access: 16 bytes of them, else two, else one, as the layout and every operand allow.
struct Widths {
  int esz, v;
  Widths(int esz, int D, int half, bool inter) : esz(esz), v(16 / esz) {
    while (v > 1 && (D % (2 * v) != 0 || (!inter && half % v != 0))) narrow();
  }
  void narrow() { v = v > 2 ? 2 : 1; }
  void rows(const void *p, int64_t st, int64_t sh) {
    while (v > 1 && (reinterpret_cast<uintptr_t>(p) % (v * esz) != 0 || st % v != 0 || sh % v != 0)) narrow();
  }
  void weights(const void *p, int64_t sh, int wsz) {  // (float32 ones in 16-byte pieces)
    auto fits = [&] {
      const int run = v * wsz < 16 ? v * wsz : 16;
      return reinterpret_cast<uintptr_t>(p) % run == 0 && sh * wsz % run == 0;
    };
    while (p != nullptr && v > 1 && !fits()) narrow();
  }
};

}  // namespace wkv
