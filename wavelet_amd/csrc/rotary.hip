// Rotary positions (gfx950): pairs of every head's leading dims turned by
// angles that grow with the token's position,
//   y_a = s (x_a cos t - x_b sin t),  y_b = s (x_b cos t + x_a sin t),
//   t = position * inv_freq[i] for pair i,
// over q and k in one launch; the dims past the turned ones are copied. With
// the sines negated it is the transpose, which is the gradient.
//
// A wave takes one token and some of its heads (all of them once there are
// tokens enough for the chip). Its lanes form the token's angles once, a pair
// each, and leave the sines and cosines in LDS for every head; a lane then
// turns units of V pairs, two 16-byte loads and two stores where the layout
// allows, some units in flight. Angles are taken in float64, in turns, and
// reduced there: float32 would lose a position of 131,072 at frequency 1 to
// 2^-7 of a radian. Sines and products are float32, one rounding to the
// type at the end.
// Bound by HBM past some thousand tokens (16,384 tokens of 40 heads of 128, bf16, in
// either layout: 61 us, 5.5 TB/s), by the launch and one round trip for a single one
// (3.4 us).
#include <cmath>

#include "wkv_common.h"

namespace wkv {

constexpr int kRotaryWaves = 4;
constexpr int kRotaryMaxPairs = WKV_ROTARY_MAX_DIM / 2;

struct RotaryRows {
  const void *x;
  void *y;
  int64_t xt, xh, yt, yh;  // strides in elements: token, head
};

struct RotaryArgs {
  RotaryRows q, k;
  const int64_t *pos;
  const double *inv_freq;
  int64_t tokens;
  int Hq, H;      // query heads; query and key heads
  int per;        // heads of a wave
  int D, half;    // head size; turned pairs
  int turned;     // units of a head that hold turned pairs only (half layout)
  FastDiv units;  // units of a head
  float scale, sign;
};

template <class T>
__device__ __forceinline__ float to_f32(T x) {
  return static_cast<float>(x);
}

// INTER: pair i is dims (2 i, 2 i + 1), else (i, i + half). A unit is V pairs
// in two runs of V elements: half apart, or (INTER, and what is only copied) half
// the units apart, so that the lanes' runs follow each other; single elements
// (V = 1) of an INTER pair are adjacent.
// FAR: rows read and written past the caches.
template <class T, int V, bool INTER, bool FAR>
__global__ __launch_bounds__(64 * kRotaryWaves) void rotary_kernel(RotaryArgs a) {
  typedef __attribute__((__vector_size__(V * sizeof(T)))) T Vec;
  __shared__ float2 turn[kRotaryWaves][kRotaryMaxPairs];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kRotaryWaves + wave;
  if (t >= a.tokens) return;  // a whole wave; nothing below waits for another
  const int h0 = blockIdx.y * a.per;
  const int heads = a.H - h0 < a.per ? a.H - h0 : a.per;
  const double p = static_cast<double>(a.pos[t]);
  for (int i = lane; i < a.half; i += 64) {
    const double x = p * a.inv_freq[i] * 0.15915494309189533577;  // 1 / 2 pi: the angle in turns
    float s, c;
    sincospif(2.f * static_cast<float>(x - rint(x)), &s, &c);
    turn[wave][i] = make_float2(c * a.scale, s * a.scale * a.sign);
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  const int n = heads * a.units.d;
  constexpr int N = FAR ? 2 : 4;  // units of a lane in flight (FAR: 4 take 8% more of the time, 1 14%)
  for (int i0 = 0; i0 < n; i0 += 64 * N) {
    Vec x0[N], x1[N];
    T *y0[N], *y1[N];
    int first[N], second[N];  // the runs' first pairs
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = i0 + 64 * k + lane;
      y0[k] = nullptr;
      if (i < n) {
        const int head = i / a.units, u = i - head * a.units.d, h = h0 + head;
        const RotaryRows &r = h < a.Hq ? a.q : a.k;
        const int hr = h < a.Hq ? h : h - a.Hq;
        int e0, e1;
        if (INTER) {
          e0 = V > 1 ? V * u : 2 * u;
          e1 = V > 1 ? V * (u + a.units.d) : 2 * u + 1;
          first[k] = e0 / 2;
          second[k] = e1 / 2;
        } else if (u < a.turned) {
          first[k] = e0 = V * u;
          e1 = e0 + a.half;
        } else {
          first[k] = a.half;
          e0 = 2 * a.half + V * (u - a.turned);
          e1 = e0 + V * (a.units.d - a.turned);
        }
        const T *x = static_cast<const T *>(r.x) + t * r.xt + hr * r.xh;
        T *y = static_cast<T *>(r.y) + t * r.yt + hr * r.yh;
        const Vec *p0 = reinterpret_cast<const Vec *>(x + e0), *p1 = reinterpret_cast<const Vec *>(x + e1);
        x0[k] = FAR ? __builtin_nontemporal_load(p0) : *p0;
        x1[k] = FAR ? __builtin_nontemporal_load(p1) : *p1;
        y0[k] = y + e0;
        y1[k] = y + e1;
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (y0[k] == nullptr) continue;
      auto turn_pair = [&](int i, T &xa, T &xb) __attribute__((always_inline)) {
        const float2 cs = turn[wave][i];
        const float fa = to_f32(xa), fb = to_f32(xb);
        xa = static_cast<T>(fa * cs.x - fb * cs.y);
        xb = static_cast<T>(fb * cs.x + fa * cs.y);
      };
      auto turn_runs = [&](int m, int w, int i) __attribute__((always_inline)) {  // elements m of x0 and w of x1
        T xa = x0[k][m], xb = x1[k][w];
        turn_pair(i, xa, xb);
        x0[k][m] = xa;
        x1[k][w] = xb;
      };
      auto turn_run = [&](Vec &x, int i0) __attribute__((always_inline)) {  // a run's adjacent pairs
#pragma unroll
        for (int v = 0; v < V / 2; ++v) {
          T xa = x[2 * v], xb = x[2 * v + 1];
          if (i0 + v < a.half) turn_pair(i0 + v, xa, xb);
          x[2 * v] = xa;
          x[2 * v + 1] = xb;
        }
      };
      if (INTER && V > 1) {
        if (first[k] < a.half) turn_run(x0[k], first[k]);  // (a run past the turned pairs' end is partly copied)
        if (second[k] < a.half) turn_run(x1[k], second[k]);
      } else if (first[k] < a.half) {
#pragma unroll
        for (int v = 0; v < V; ++v) turn_runs(v, v, first[k] + v);
      }
      if (FAR) {
        __builtin_nontemporal_store(x0[k], reinterpret_cast<Vec *>(y0[k]));
        __builtin_nontemporal_store(x1[k], reinterpret_cast<Vec *>(y1[k]));
      } else {
        *reinterpret_cast<Vec *>(y0[k]) = x0[k];
        *reinterpret_cast<Vec *>(y1[k]) = x1[k];
      }
    }
  }
}

// Elements per access: the widest up to 16 bytes that the layout allows.
static int rotary_width(int esz, int D, int half, bool inter, const RotaryRows *r, int n) {
  for (int v = 16 / esz; v > 1; v /= 2) {
    bool fits = D % (2 * v) == 0 && (inter || half % v == 0);
    for (int i = 0; i < n && fits; ++i)
      fits = reinterpret_cast<uintptr_t>(r[i].x) % (v * esz) == 0 && reinterpret_cast<uintptr_t>(r[i].y) % (v * esz) == 0 &&
             r[i].xt % v == 0 && r[i].xh % v == 0 && r[i].yt % v == 0 && r[i].yh % v == 0;
    if (fits) return v;
  }
  return 1;
}

template <class T, bool INTER>
static void launch_rotary(const RotaryArgs &a, int v, bool far, dim3 grid, hipStream_t s) {
  constexpr int B = 64 * kRotaryWaves, W = 16 / sizeof(T);
  if (v == W && far) return rotary_kernel<T, W, INTER, true><<<grid, B, 0, s>>>(a);
  if (v == W) return rotary_kernel<T, W, INTER, false><<<grid, B, 0, s>>>(a);
  if (W > 4 && v == 4) return rotary_kernel<T, 4, INTER, false><<<grid, B, 0, s>>>(a);  // (narrower: never far)
  if (v == 2) return rotary_kernel<T, 2, INTER, false><<<grid, B, 0, s>>>(a);
  rotary_kernel<T, 1, INTER, false><<<grid, B, 0, s>>>(a);
}

}  // namespace wkv

using namespace wkv;

extern "C" int wkv_rotary(int32_t dtype, const void *q, int64_t q_stride_t, int64_t q_stride_h, void *q_out,
                          int64_t qo_stride_t, int64_t qo_stride_h, int32_t num_q_heads, const void *k,
                          int64_t k_stride_t, int64_t k_stride_h, void *k_out, int64_t ko_stride_t,
                          int64_t ko_stride_h, int32_t num_k_heads, int32_t head_dim, const int64_t *positions,
                          const double *inv_freq, int32_t rotary_dim, int32_t interleaved, int32_t inverse, float scale,
                          int64_t num_tokens, void *stream) {
  WKV_CHECK_ARG(dtype >= 0 && dtype <= 2, "dtype must be 0 (fp32), 1 (bf16) or 2 (fp16) (got %d)", dtype);
  WKV_CHECK_ARG(num_tokens >= 0 && num_tokens <= INT32_MAX, "num_tokens must be in [0, 2^31) (got %lld)",
                (long long)num_tokens);
  WKV_CHECK_ARG(num_q_heads >= 0 && num_k_heads >= 0 && num_q_heads <= 65535 && num_k_heads <= 65535,
                "head counts must be in [0, 65535]");
  WKV_CHECK_ARG(head_dim > 0 && head_dim % 2 == 0 && head_dim <= WKV_ROTARY_MAX_DIM,
                "head_dim must be even and in [2, %d] (got %d)", WKV_ROTARY_MAX_DIM, head_dim);
  WKV_CHECK_ARG(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim,
                "rotary_dim must be even and in [2, head_dim] (got %d)", rotary_dim);
  WKV_CHECK_ARG(std::isfinite(scale), "scale must be finite");
  const int H = num_q_heads + num_k_heads;
  if (num_tokens == 0 || H == 0) return WKV_OK;
  const int esz = dtype == 0 ? 4 : 2;
  auto rows_ok = [&](const void *x, const void *y, int heads) {
    return heads == 0 || (x != nullptr && y != nullptr && reinterpret_cast<uintptr_t>(x) % esz == 0 &&
                          reinterpret_cast<uintptr_t>(y) % esz == 0);
  };
  WKV_CHECK_ARG(rows_ok(q, q_out, num_q_heads) && rows_ok(k, k_out, num_k_heads),
                "q / k and their outputs must be non-NULL and aligned to their elements");
  WKV_CHECK_ARG(q_stride_t >= 0 && q_stride_h >= 0 && qo_stride_t >= 0 && qo_stride_h >= 0 && k_stride_t >= 0 &&
                    k_stride_h >= 0 && ko_stride_t >= 0 && ko_stride_h >= 0,
                "strides must be non-negative");
  WKV_CHECK_ARG(positions != nullptr && reinterpret_cast<uintptr_t>(positions) % 8 == 0 && inv_freq != nullptr &&
                    reinterpret_cast<uintptr_t>(inv_freq) % 8 == 0,
                "positions and inv_freq must be non-NULL, int64 and float64");
  RotaryArgs a{};
  a.q = RotaryRows{q, q_out, q_stride_t, q_stride_h, qo_stride_t, qo_stride_h};
  a.k = RotaryRows{k, k_out, k_stride_t, k_stride_h, ko_stride_t, ko_stride_h};
  a.pos = positions;
  a.inv_freq = inv_freq;
  a.tokens = num_tokens;
  a.Hq = num_q_heads;
  a.H = H;
  a.D = head_dim;
  a.half = rotary_dim / 2;
  a.scale = scale;
  a.sign = inverse ? -1.f : 1.f;
  const bool inter = interleaved != 0;
  const RotaryRows rows[2] = {num_q_heads ? a.q : a.k, num_k_heads ? a.k : a.q};
  const int v = rotary_width(esz, head_dim, a.half, inter, rows, 2);
  a.turned = a.half / v;
  const int units = head_dim / (2 * v);
  a.units = fast_div(units);
  // All heads of a token in one wave share its angles; with too few tokens for
  // the chip (four waves per SIMD) they are dealt over more waves, down to a
  // round of 64 units each.
  const int least = units >= 64 ? 1 : 64 / units;
  const int64_t want = (4096 + num_tokens - 1) / num_tokens;
  const int most = (H + least - 1) / least;
  const int split = want < most ? static_cast<int>(want) : most;
  a.per = (H + split - 1) / split;
  const dim3 grid(static_cast<unsigned>((num_tokens + kRotaryWaves - 1) / kRotaryWaves),
                  static_cast<unsigned>((H + a.per - 1) / a.per));
  // Rows far larger than the caches go past them (32 query and 8 key heads of 128,
  // bf16, near / far: 4,096 tokens 16.0 / 18.6 us, 16,384 into new memory 72 / 61, 32,768
  // 131 / 117; stored near, 16,384 take 65 into new memory and 55 into memory just written).
  const bool far = static_cast<int64_t>(num_tokens) * H * head_dim * esz >= (64 << 20);
  auto s = static_cast<hipStream_t>(stream);
  if (dtype == 0) {
    if (inter) launch_rotary<float, true>(a, v, far, grid, s); else launch_rotary<float, false>(a, v, far, grid, s);
  } else if (dtype == 1) {
    if (inter) launch_rotary<__bf16, true>(a, v, far, grid, s); else launch_rotary<__bf16, false>(a, v, far, grid, s);
  } else {
    if (inter) launch_rotary<_Float16, true>(a, v, far, grid, s); else launch_rotary<_Float16, false>(a, v, far, grid, s);
  }
  WKV_CHECK_LAUNCH("rotary");
  return WKV_OK;
}
