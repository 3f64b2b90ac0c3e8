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
// sum of squares is a butterfly over the group. The groups of a wave take a few tokens and
// walk their heads: a lane's token and unit stay the same, so that its
// angles and weights are formed once, as the products that y is linear in x by,
//   y_a = (x_a r) (w_a c) - (x_b r) (w_b s),  y_b = (x_b r) (w_b c) + (x_a r) (w_a s),
// and a value costs some 14 vector instructions, the angles' among them (counted for 16,384 tokens of 32 + 8 heads
// of 128).
#pragma once

#include <cmath>
#include <type_traits>

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

// The position of pair i at token t. A pair of an axis that is not there stays (0).
__device__ __forceinline__ int64_t position_at(const Angles &a, int64_t t, int i) {
  if (a.axes == nullptr) return a.pos[t];  // uniform
  const int ax = a.axes[i];
  return static_cast<unsigned>(ax) < static_cast<unsigned>(a.num_axes) ? a.pos[ax * a.axis_stride + t] : 0;
}

// Cosine and sine of a position's angle, times the scale: the angle in turns and its distance from the
// nearest quarter of one in float64, then the Taylor series of that distance, at most pi / 4: to z^4 (sine)
// and z^5 (cosine) of its square z, whose next terms are below 2^-28 of it and 2^-32. Off by at most 1.3 x
// 2^-24 (a float32 of half a turn alone by 1.6), 0.3 in the mean, which decides how often a key's last bit,
// and its code, is the exact one's. That is for angles below 2^27; from there on float64's own rounding of
// the angle, some 2^-52 of it, is the larger part (3.6 x 2^-24 in all at 2^30). The series in float64, rounded once,
// costs more than it gives: an fp8 append of 8,386 tokens of 28/4 heads 45 us in the place of 38.
__device__ __forceinline__ float2 angle_of(const Angles &a, int64_t pos, double freq) {
  const double x = static_cast<double>(pos) * freq * 0.15915494309189533577;  // 1 / 2 pi
  const double y = 4. * (x - rint(x)), n = rint(y);
  const float r = static_cast<float>((y - n) * 1.57079632679489661923), z = r * r;
  float p = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);  // 1 / 9!, -1 / 7!
  p = __builtin_fmaf(z, p, 8.3333333e-3f);
  p = __builtin_fmaf(z, p, -1.6666667e-1f);
  const float s0 = __builtin_fmaf(r * z, p, r);
  float q = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);  // -1 / 10!, 1 / 8!
  q = __builtin_fmaf(z, q, -1.3888889e-3f);
  q = __builtin_fmaf(z, q, 4.1666667e-2f);
  q = __builtin_fmaf(z, q, -0.5f);
  const float c0 = __builtin_fmaf(z, q, 1.f);
  const int k = static_cast<int>(n);  // quarters, -2 to 2
  const float c = k & 1 ? s0 : c0, s = k & 1 ? c0 : s0;
  return make_float2((k + 1) & 2 ? -c * a.scale : c * a.scale, (k & 2 ? -s : s) * a.scale * a.sign);
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

// The sum over a group of 2^log_lanes lanes, the same in each. LL: log_lanes as a constant (-1: it is none).
template <int LL = -1>
__device__ __forceinline__ float group_sum(float v, int log_lanes) {
  if (LL >= 0) log_lanes = LL;
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

// Pair p of a unit, as its elements of the runs x0 and x1.
template <int V, bool INTER>
__device__ __forceinline__ float &pair_a(int p, float *x0, float *x1) {
  return INTER && V > 1 ? (p < V / 2 ? x0[2 * p] : x1[2 * p - V]) : x0[p];
}
template <int V, bool INTER>
__device__ __forceinline__ float &pair_b(int p, float *x0, float *x1) {
  return INTER && V > 1 ? (p < V / 2 ? x0[2 * p + 1] : x1[2 * p - V + 1]) : x1[p];
}

// A unit's cosines and sines; pairs that are not turned: (1, 0), and their bits of `live` are clear.
template <int V>
struct UnitTurn {
  float c[V], s[V];
  uint32_t live;
};

template <int V, bool INTER>
__device__ __forceinline__ void unit_turn(const float2 *turn, int half, bool all, int e0, int e1, UnitTurn<V> &t) {
  auto pair = [&](int p) { return INTER && V > 1 ? (p < V / 2 ? e0 / 2 + p : e1 / 2 + p - V / 2) : INTER ? e0 / 2 : e0 + p; };
  t.live = (1u << V) - 1u;
  if (all) {  // uniform
#pragma unroll
    for (int p = 0; p < V; ++p) {
      const float2 cs = turn[pair(p)];
      t.c[p] = cs.x;
      t.s[p] = cs.y;
    }
    return;
  }
#pragma unroll
  for (int p = 0; p < V; ++p) {
    const int i = pair(p);
    const float2 cs = half > 0 ? turn[i < half ? i : half - 1] : make_float2(1.f, 0.f);
    t.c[p] = i < half ? cs.x : 1.f;
    t.s[p] = i < half ? cs.y : 0.f;
    if (i >= half) t.live &= ~(1u << p);
  }
}

// The products of a unit's weights, cosines and sines.
template <int V>
struct UnitCoef {
  float ac[V], bs[V], bc[V], as[V];
};

template <int V, bool INTER>
__device__ __forceinline__ void unit_coef(const UnitTurn<V> &t, float *w0, float *w1, UnitCoef<V> &k) {
#pragma unroll
  for (int p = 0; p < V; ++p) {
    const float a = pair_a<V, INTER>(p, w0, w1), b = pair_b<V, INTER>(p, w0, w1);
    k.ac[p] = a * t.c[p];
    k.bs[p] = b * t.s[p];
    k.bc[p] = b * t.c[p];
    k.as[p] = a * t.s[p];
  }
}

// A unit of x times inv, normed and turned in place. all: every pair is turned (else an infinity's pair would
// take it in as a NaN).
template <int V, bool INTER>
__device__ __forceinline__ void unit_apply(const UnitCoef<V> &k, uint32_t live, bool all, float inv, float *x0, float *x1) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    x0[v] *= inv;
    x1[v] *= inv;
  }
  auto turn = [&](auto whole) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < V; ++p) {
      float &a = pair_a<V, INTER>(p, x0, x1), &b = pair_b<V, INTER>(p, x0, x1);
      float t = b * k.bs[p], u = a * k.as[p];
      if (!decltype(whole)::value && !(live >> p & 1)) t = u = 0.f;
      a = __builtin_fmaf(a, k.ac[p], -t);
      b = __builtin_fmaf(b, k.bc[p], u);
    }
  };
  if (all)
    turn(std::true_type{});
  else
    turn(std::false_type{});
}

// unit_turn, unit_coef and unit_apply of one row, pair by pair: the same values from fewer registers.
template <int V, bool INTER>
__device__ __forceinline__ void unit_once(const float2 *turn, int half, bool all, int e0, int e1, const float *w0, const float *w1,
                                          float inv, float *x0, float *x1) {
  auto pair = [&](int p) { return INTER && V > 1 ? (p < V / 2 ? e0 / 2 + p : e1 / 2 + p - V / 2) : INTER ? e0 / 2 : e0 + p; };
#pragma unroll
  for (int p = 0; p < V; ++p) {
    const int i = pair(p);
    float2 cs = make_float2(1.f, 0.f);
    if (half > 0) cs = turn[all || i < half ? i : 0];
    const bool live = all || i < half;
    if (!live) cs = make_float2(1.f, 0.f);
    float &a = pair_a<V, INTER>(p, x0, x1), &b = pair_b<V, INTER>(p, x0, x1);
    const float wa = pair_a<V, INTER>(p, const_cast<float *>(w0), const_cast<float *>(w1));
    const float wb = pair_b<V, INTER>(p, const_cast<float *>(w0), const_cast<float *>(w1));
    const float xa = a * inv, xb = b * inv;
    float t = xb * (wb * cs.y), u = xa * (wa * cs.y);
    if (!live) t = u = 0.f;
    a = __builtin_fmaf(xa, wa * cs.x, -t);
    b = __builtin_fmaf(xb, wb * cs.x, u);
  }
}

// A unit turned alone, without weights (a gradient's, by the transpose's angles).
template <int V, bool INTER>
__device__ __forceinline__ void unit_back(const UnitTurn<V> &t, bool all, float *x0, float *x1) {
  auto turn = [&](auto whole) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < V; ++p) {
      float &a = pair_a<V, INTER>(p, x0, x1), &b = pair_b<V, INTER>(p, x0, x1);
      float u = b * t.s[p], v = a * t.s[p];
      if (!decltype(whole)::value && !(t.live >> p & 1)) u = v = 0.f;
      a = __builtin_fmaf(a, t.c[p], -u);
      b = __builtin_fmaf(b, t.c[p], v);
    }
  };
  if (all)
    turn(std::true_type{});
  else
    turn(std::false_type{});
}

// The angles of tokens t0 .. t0 + nt - 1, thread `tid` of `threads`, while there are as many B at a time:
// their positions and frequencies are all requested before the first is used.
template <int B>
__device__ __forceinline__ void angles_of(const Angles &a, int64_t t0, int nt, int tid, int threads, float2 *turn) {
  const int n = nt * a.half.d;
  int i = tid;
  if constexpr (B > 1) {
    for (; i - tid + B * threads <= n; i += B * threads) {  // uniform
      int64_t pos[B];
      double freq[B];
#pragma unroll
      for (int k = 0; k < B; ++k) {
        const int t = (i + threads * k) / a.half, p = i + threads * k - t * a.half.d;
        pos[k] = position_at(a, t0 + t, p);
        freq[k] = a.inv_freq[p];
      }
#pragma unroll
      for (int k = 0; k < B; ++k) turn[i + threads * k] = angle_of(a, pos[k], freq[k]);
    }
  }
  for (; i < n; i += threads) {
    const int t = i / a.half, p = i - t * a.half.d;
    turn[i] = angle_of(a, position_at(a, t0 + t, p), a.inv_freq[p]);
  }
}

// The same by one wave, for its own reads.
template <int B = 1>
__device__ __forceinline__ void wave_angles(const Angles &a, int64_t t0, int nt, float2 *turn) {
  angles_of<B>(a, t0, nt, threadIdx.x & 63, 64, turn);
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A kind of heads of one token, as a lane sees them.
template <class T>
struct HeadsOf {
  const T *x;      // head 0 (of those that the wave takes)
  int64_t xh;      // elements between heads
  T *y;
  int64_t yh;
  int piece;       // 0: y is a row; else element e is at (e / 8) piece + e % 8 (a cache's keys)
  const void *w;   // the weights of head 0 (nullptr: ones)
  int64_t ws;      // between heads; not 0: each head has its own
};

// A kind of heads in a launch.
struct Kind {
  HeadRows s;
  const void *w;
  int64_t ws;
  int heads;
  int log_tg, per;  // KindGrid
  FastDiv splits;
};

// Which tokens and heads wave `wave` of workgroup wg of a kind takes, and where its lane stands.
struct WaveTile {
  int64_t t0;        // the wave's first token
  int tokens;        // of it; 0: none
  int h0, heads;     // its heads
  int t, group;      // the lane's token of them, its group's number among the token's
  bool there;        // there is such a token
};

__device__ __forceinline__ WaveTile wave_tile(const Kind &k, const RowUnits &r, int64_t tokens, int wg, int wave) {
  WaveTile w;
  const int x = wg / k.splits, split = wg - x * k.splits.d, tg = 1 << k.log_tg;
  w.t0 = (static_cast<int64_t>(x) * 4 + wave) << k.log_tg;
  w.tokens = w.t0 >= tokens ? 0 : tokens - w.t0 < tg ? static_cast<int>(tokens - w.t0) : tg;
  w.h0 = split * k.per;
  w.heads = k.heads - w.h0 < k.per ? k.heads - w.h0 : k.per;
  const int g = (threadIdx.x & 63) >> r.log_lanes;
  w.t = g & (tg - 1);
  w.group = g >> k.log_tg;
  w.there = w.t < w.tokens;
  if (!w.there) w.t = 0;
  return w;
}

// The heads first, first + step, .. below `heads` of the lane's token (there: it has one), normed (if
// norm.on) and turned by turn[], the next one in flight meanwhile; ready(): called once the
// first is, before turn[] is read. EACH: each head's own weights.
template <class T, int V, bool INTER, int U, bool FAR, bool NEAR_STORE, bool EACH, int LL, class Ready>
__device__ __forceinline__ void norm_turn_heads(const RowUnits &ru, const HeadNorm &norm, const float2 *turn, bool there,
                                                int first, int step, int heads, const HeadsOf<T> &of, Ready ready) {
  typedef typename VecOf<T, V>::type Vec;
  const int lanes = 1 << (LL >= 0 ? LL : ru.log_lanes), u0 = threadIdx.x & (lanes - 1);
  const float inv_d = 1.f / static_cast<float>(ru.D);
  const bool all = 2 * ru.half == ru.D;
  int e0[U], e1[U];
  bool mine[U];
#pragma unroll
  for (int j = 0; j < U; ++j) {
    const int u = u0 + lanes * j;
    mine[j] = there && u < ru.units;
    e0[j] = e1[j] = 0;
    if (u < ru.units) unit_runs<V, INTER>(ru, u, e0[j], e1[j]);
  }
  Vec n0[U], n1[U];
  auto load = [&](int h) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      n0[j] = n1[j] = Vec{};
      if (mine[j] && h < heads) {
        const Vec *p0 = reinterpret_cast<const Vec *>(of.x + h * of.xh + e0[j]);
        const Vec *p1 = reinterpret_cast<const Vec *>(of.x + h * of.xh + e1[j]);
        n0[j] = FAR ? __builtin_nontemporal_load(p0) : *p0;
        n1[j] = FAR ? __builtin_nontemporal_load(p1) : *p1;
      }
    }
  };
  load(first);
  float w0[U][V], w1[U][V];
  if (!EACH) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      load_weights<T, V>(norm, of.w, e0[j], w0[j]);
      load_weights<T, V>(norm, of.w, e1[j], w1[j]);
    }
  }
  ready();
  UnitTurn<V> t[U];
  UnitCoef<V> coef[U];
#pragma unroll
  for (int j = 0; j < U; ++j) {
    unit_turn<V, INTER>(turn, ru.half, all, e0[j], e1[j], t[j]);
    if (!EACH) unit_coef<V, INTER>(t[j], w0[j], w1[j], coef[j]);
  }
  for (int hb = 0; hb < heads; hb += step) {  // uniform; the lane's row is hb + first
    Vec x0[U], x1[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      x0[j] = n0[j];
      x1[j] = n1[j];
    }
    if (hb + step < heads) load(hb + step + first);
    const int h = hb + first;
    float f0[U][V], f1[U][V], ss = 0.f;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      widen<V, T>(x0[j], f0[j]);
      widen<V, T>(x1[j], f1[j]);
#pragma unroll
      for (int v = 0; v < V; ++v) ss = __builtin_fmaf(f0[j][v], f0[j][v], __builtin_fmaf(f1[j][v], f1[j][v], ss));
    }
    ss = group_sum<LL>(ss, ru.log_lanes);
    const float inv = norm.on ? __builtin_amdgcn_rsqf(__builtin_fmaf(ss, inv_d, norm.eps)) : 1.f;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (EACH) {
        const int64_t wh = h < heads ? h * of.ws : 0;
        load_weights<T, V>(norm, of.w, wh + e0[j], w0[j]);
        load_weights<T, V>(norm, of.w, wh + e1[j], w1[j]);
        unit_coef<V, INTER>(t[j], w0[j], w1[j], coef[j]);
      }
      unit_apply<V, INTER>(coef[j], t[j].live, all, inv, f0[j], f1[j]);
      if (mine[j] && h < heads) {
        Vec o0, o1;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          o0[v] = static_cast<T>(f0[j][v]);
          o1[v] = static_cast<T>(f1[j][v]);
        }
        T *y = of.y + h * of.yh;
        const int i0 = of.piece == 0 ? e0[j] : (e0[j] >> 3) * of.piece + (e0[j] & 7);
        const int i1 = of.piece == 0 ? e1[j] : (e1[j] >> 3) * of.piece + (e1[j] & 7);
        if (FAR && !NEAR_STORE) {
          __builtin_nontemporal_store(o0, reinterpret_cast<Vec *>(y + i0));
          __builtin_nontemporal_store(o1, reinterpret_cast<Vec *>(y + i1));
        } else {
          *reinterpret_cast<Vec *>(y + i0) = o0;
          *reinterpret_cast<Vec *>(y + i1) = o1;
        }
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

// Workgroups of a launch: 2^32 work items.
constexpr int64_t kMaxWorkgroups = (1 << 24) - 1;

// Waves over the tokens and heads of a kind, four a workgroup: a token a wave (its heads lie together;
// by_token: as many as the wave's groups, whose stores of one head then lie together in a cache), and with
// too few tokens for the chip the heads dealt over more waves, down to a round of the wave's groups below
// 4,096 waves (four a SIMD), to two rounds below 16,384 (4,696 tokens of 128 heads of 64: 38 us, 45 a
// wave a token; 8,191 of 16 heads of 128, two rounds, lose 1 us in halves).
struct KindGrid {
  int log_tg = 0, per = 1, splits = 1;
  int64_t waves = 0, wgs = 0;
  KindGrid(int64_t tokens, int heads, int log_lanes, bool by_token) {
    if (tokens <= 0 || heads <= 0) return;
    const int log_groups = 6 - log_lanes;
    while (by_token && log_tg < log_groups && (tokens >> (log_tg + 1)) * heads >= 4096) ++log_tg;
    waves = ((tokens - 1) >> log_tg) + 1;
    const int step = (1 << log_groups) >> log_tg, rounds = (heads + step - 1) / step;
    auto share = [&](int64_t want, int most) {
      const int64_t n = (want + waves - 1) / waves;
      return static_cast<int>(n < most ? n : most);
    };
    const int few = share(4096, rounds), many = by_token ? 1 : share(16384, rounds / 2), n = few > many ? few : many;
    per = (rounds + n - 1) / n * step;
    splits = (heads + per - 1) / per;
    wgs = (waves + 3) / 4 * splits;
  }
};

// The elements of an access: 16 bytes of them, else two, else one, as the layout and every operand allow. The
// narrow ones are for what models seldom have, half a rotation of no multiple of 16 bytes, and unaligned rows: 16,384
// tokens of 40 heads of 128, bf16, half 64 / 46 / 45: 65 / 85 / 112 us; with the append 81 / 106 / 156.
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
