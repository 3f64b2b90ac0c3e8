// Attention of a tree of drafted tokens over the paged cache (gfx950).
//
// Sequence b brings n_b drafted tokens (the last n_b of its L_b = seq_lens[b])
// and every one of its G query heads per KV head: n_b G rows of one KV head that
// read the same keys. All rows see the context's keys; of the drafted tokens'
// keys a row sees those whose bit its mask sets.
//
// Work: the rows of one (sequence, KV head), node by node with the G heads of a
// node together, are taken 32 at a time by a wave (a unit: the columns of its
// 32x32x16 MFMAs), four units to a workgroup, so that up to 128 rows share one
// read of the keys. 64-key steps are copied to LDS by LDS-DMA, a 16-key tile
// by each wave, NS steps in flight; a wave without rows only copies. Long
// contexts are cut into chunks of whole steps over workgroups (each sequence's
// steps spread evenly over its chunks), whose fp32 partials a second kernel
// merges by log-sum-exp.
// Bound by reading K and V once: at 128 rows a step's 64 MFMAs of a SIMD pair
// take as long as its 32 KB at the chip's read rate, below that the memory is
// what lasts.
//
// fp8 caches stay in their codes in LDS; a wave widens its operands as it reads
// them (exact) and applies the power-of-two scales to the scores (K) and the
// probabilities (V).
//
// Masked keys: scores are -inf after scaling (a step's window of the row's mask
// as 64 bits), so that neither the scale's sign nor a NaN key matters. A masked
// probability is 0, but 0 times a V that is not finite is NaN: in steps that
// mask anything a tile with such a V is added key by key, to the rows that see the key.
#include <cmath>

#include "gqa_tiles.h"
#include "lds_dma.h"

namespace wkv {

constexpr int kTreeWaves = 4;
constexpr int kTreeRows = 32 * kTreeWaves;  // rows of a workgroup
constexpr int kTreeCus = 256;

struct TreeArgs {
  const uint8_t *kc, *vc;
  const float *ksc, *vsc;
  const uint16_t *q;
  int64_t q_st, q_sh;
  uint16_t *out;
  int64_t o_st, o_sh;
  const int32_t *cu_q, *seq_lens, *bt;
  int64_t bt_stride;
  const int64_t *mask;
  int words;
  int Mb, max_seq, Hkv, G, BS, nb;
  FastDiv by_BS, by_G, by_Hkv, by_chunks;
  int items;        // (sequence, KV head) x chunks
  int chunks;       // most chunks of a sequence
  int chunk_steps;  // most 64-key steps of one
  int units;        // units per (sequence, KV head) at the longest query
  float scale_log2;
  float *part;
  const float *sinks;
};

// The chunks of a sequence of L tokens: as many as its steps need at chunk_steps
// each, the steps spread evenly over them.
struct TreeChunks {
  int n, per;
};
__device__ __forceinline__ TreeChunks tree_chunks(int L, int chunk_steps, int steps) {
  TreeChunks c;
  c.n = (steps + chunk_steps - 1) / chunk_steps;
  c.per = c.n > 0 ? (steps + c.n - 1) / c.n : 0;
  c.n = __builtin_amdgcn_readfirstlane(c.n);
  c.per = __builtin_amdgcn_readfirstlane(c.per);
  return c;
}

// A unit's partial of a chunk: D / 32 x 4 runs of 64 lanes x 4 fp32 (the output
// accumulators as the lanes hold them), then the 32 rows' reference maxima (log2
// domain) and sums.
template <int D>
constexpr int tree_part_floats() {
  return 32 * D + 64;
}

template <int D, bool FP8>
constexpr int tree_steps_in_lds() {
  return (FP8 ? 1 : 2) * D >= 256 ? 2 : 4;
}

template <int D, bool FP8, int NS>
__global__ __launch_bounds__(64 * kTreeWaves, 2) void tree_gqa_kernel(TreeArgs a) {
  constexpr int ESZ = FP8 ? 1 : 2;
  constexpr int TB = D * 16 * ESZ;  // bytes of a 16-key tile's K, and of its V
  constexpr int NC = TB / 1024;     // 1 KB copies of each
  constexpr int DV = D / 64;        // bf16 V copies per token octet
  __shared__ __attribute__((aligned(16))) uint8_t ldsk[NS * 4 * TB];
  __shared__ __attribute__((aligned(16))) uint8_t ldsv[NS * 4 * TB];
  __shared__ __attribute__((aligned(16))) int s_ok[NS][4];          // the tile holds keys
  __shared__ __attribute__((aligned(16))) float s_ks[NS][4], s_vs[NS][4];  // fp8: its block's scales
  __shared__ uint64_t s_mask[kTreeRows][WKV_TREE_MAX_WORDS];
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63, n = lane & 31, hh = lane >> 5;

  // The row groups of one item stand eight workgroups apart: on one XCD, whose
  // L2 then serves their keys.
  const int item = static_cast<int>(blockIdx.y) * 8 + static_cast<int>(blockIdx.x & 7);
  const int rb = static_cast<int>(blockIdx.x >> 3);
  if (item >= a.items) return;
  const int bc = item / a.by_Hkv, kvh = item - bc * a.Hkv;
  const int b = bc / a.by_chunks, chunk = bc - b * a.chunks;
  const int q0 = a.cu_q[b], qlen = a.cu_q[b + 1] - q0;
  int L = a.seq_lens[b];
  L = L < a.max_seq ? L : a.max_seq;
  const int G = a.G;
  const int rows = qlen * G;
  if (qlen <= 0 || rb * kTreeRows >= rows) return;
  const int unit = rb * kTreeWaves + wave;
  const bool active = 32 * unit < rows;  // uniform
  const int row = 32 * unit + n;
  const bool has_row = row < rows;
  const int node = has_row ? row / a.by_G : 0;
  const int h = kvh * G + (has_row ? row - node * G : 0);
  uint16_t *const op = a.out + static_cast<int64_t>(q0 + node) * a.o_st + static_cast<int64_t>(h) * a.o_sh;
  if (L <= 0) {  // nothing to attend to
    if (chunk == 0 && has_row)
#pragma unroll
      for (int d = 0; d < D; d += 8) *reinterpret_cast<u32x2 *>(op + d + 4 * hh) = u32x2{0u, 0u};
    return;
  }
  const int all_steps = (L + 63) >> 6;
  const TreeChunks tc = tree_chunks(L, a.chunk_steps, all_steps);
  if (chunk >= tc.n) return;  // the whole workgroup
  const int s0 = chunk * tc.per;
  const int s1 = s0 + tc.per < all_steps ? s0 + tc.per : all_steps;
  const int ctx = L - qlen;  // the first drafted token's position

  // Q^T operand j: lane l holds d = 16 j + 8 (l / 32) .. + 7 of row l % 32.
  bf16x8 qb[D / 16];
  {
    const uint16_t *qp = a.q + static_cast<int64_t>(q0 + node) * a.q_st + static_cast<int64_t>(h) * a.q_sh;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      u32x4 w = *reinterpret_cast<const u32x4 *>(qp + 16 * j + 8 * hh);
      if (!has_row) w = u32x4{0u, 0u, 0u, 0u};
      qb[j] = __builtin_bit_cast(bf16x8, w);
    }
  }
  if (64 * s1 > ctx && hh == 0) {  // (read by this wave's own lanes)
    const int64_t *mp = a.mask + static_cast<int64_t>(q0 + node) * a.words;
#pragma unroll
    for (int w = 0; w < WKV_TREE_MAX_WORDS; ++w)
      s_mask[32 * wave + n][w] = has_row && w < a.words ? static_cast<uint64_t>(mp[w]) : 0ull;
  }

  floatx16 o[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[c][r] = 0.f;
  float m_ref = -INFINITY, l_part = 0.f;  // reference maximum (-inf until a key is seen), this lane's share of the sum

  // Copies. Piece p = 64 k + l of a tile's K or V goes to LDS offset 16 p. K: chunk p / 16,
  // token p % 16, as the cache holds it. bf16 V: row p % D of token octet p / D;
  // fp8 V: row p.
  const int BS = a.BS, region = D * BS * ESZ;
  const uint32_t lane_k = static_cast<uint32_t>(((lane >> 4) * BS + (lane & 15)) * 16);
  const uint32_t lane_v = static_cast<uint32_t>(lane * BS * ESZ);
  const uint32_t ldsk0 = lds_addr(ldsk), ldsv0 = lds_addr(ldsv);
  const int32_t *const btrow = a.bt + b * a.bt_stride;
  const int key_w = 64 * s0 + 16 * wave;
  int bix = key_w / a.by_BS;
  int o0 = key_w - bix * BS;
  const int dbix = 64 / a.by_BS, do0 = 64 - dbix * BS;
  int wbase = bix;  // the window: lane i holds the id of block wbase + i
  int win = load_i32_drained(btrow, wbase + lane, a.Mb);
  uint32_t issued = 0;  // a bit per step, the last one lowest: this wave copied a tile of it
  auto issue = [&](int s, int slot) {
    issued <<= 1;
    bool ok = s < s1 && 64 * s + 16 * wave < L;  // uniform
    if (ok) {
      if (bix - wbase >= 64) {  // at most once per 64 blocks (its wait drains the copies in flight)
        wbase = bix;
        win = load_i32_drained(btrow, wbase + lane, a.Mb);
      }
      const int blk = __builtin_amdgcn_readlane(win, bix - wbase);
      ok = blk >= 0 && blk < a.nb;
      if (ok) {
        const int64_t rb_ = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(blk * a.Hkv + kvh)) *
                                                 static_cast<uint32_t>(region));
        if constexpr (FP8) {
          const float ks = load_scalar(a.ksc + blk * a.Hkv + kvh), vs = load_scalar(a.vsc + blk * a.Hkv + kvh);
          if (lane == 0) {
            s_ks[slot][wave] = ks;
            s_vs[slot][wave] = vs;
          }
        }
        uint32_t kst = static_cast<uint32_t>(64 * BS), vst = static_cast<uint32_t>((FP8 ? 64 : 128) * BS);
        asm volatile("" : "+s"(kst), "+s"(vst));
        const __amdgpu_buffer_rsrc_t kr =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(a.kc + rb_ + o0 * 16), 0, region, kRawBufferWord3);
        const uint32_t tile = static_cast<uint32_t>((4 * slot + wave) * TB);
        buffer_copy16_run_to_lds<NC>(kr, lane_k, kst - 1024u, ldsk0 + tile);
        const __amdgpu_buffer_rsrc_t vr =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(a.vc + rb_ + o0 * ESZ), 0, region, kRawBufferWord3);
#pragma unroll
        for (int k = 0; k < NC; ++k)
          buffer_copy16_to_lds(vr, lane_v, FP8 ? vst * k : vst * (k % DV) + 16 * (k / DV), ldsv0 + tile + 1024 * k);
        issued |= 1;
      }
    }
    if (lane == 0) s_ok[slot][wave] = ok ? 1 : 0;
    o0 += do0;
    bix += dbix;
    if (o0 >= BS) {
      o0 -= BS;
      ++bix;
    }
  };
  // Until the copies of all but the last NS - 2 steps issued have landed (this wave's).
  auto wait_step = [&]() {
    const int later = __builtin_popcount(issued & ((1u << (NS - 2)) - 1u));  // uniform
    if (NS > 2 && later >= 1) {
      if (NS > 3 && later >= 2)
        wait_vmcnt<(NS > 3 ? 4 * NC : 0)>();
      else
        wait_vmcnt<(NS > 2 ? 2 * NC : 0)>();
    } else {
      wait_vmcnt<0>();
    }
  };

  // Row i of a 32-key half's S^T carries key kperm(i), so that score r of lane
  // l is key 16 (r / 8) + 8 (l / 32) + r % 8 of the half: the PV operand as it stands.
  const int kn = (n & 16) | (((n >> 2) & 3) == 1 ? (n & 3) + 8 : ((n >> 2) & 3) == 2 ? (n & 3) + 4 : (n & 15));
  const bf16x2 ones = __builtin_bit_cast(bf16x2, 0x3F803F80u);

  // V operand: row 32 c + n, the tokens 8 hh .. + 7 of tile t of a slot, as bf16.
  auto v_operand = [&](int slot, int t, int c) {
    const uint8_t *lv = ldsv + (4 * slot + t) * TB;
    if constexpr (FP8) {
      const u32x2 w = *reinterpret_cast<const u32x2 *>(lv + (32 * c + n) * 16 + 8 * hh);
      return __builtin_bit_cast(u32x4, fp8x8_to_bf16x8(w[0], w[1]));
    } else {
      return *reinterpret_cast<const u32x4 *>(lv + (hh * D + 32 * c + n) * 16);
    }
  };
  // V of row d, token e of tile t
  auto v_value = [&](int slot, int t, int d, int e) {
    const uint8_t *lv = ldsv + (4 * slot + t) * TB;
    if constexpr (FP8)
      return __builtin_amdgcn_cvt_f32_fp8(lv[d * 16 + e], 0);
    else
      return bf16_bits_to_f32(*reinterpret_cast<const uint16_t *>(lv + ((e >> 3) * D + d) * 16 + 2 * (e & 7)));
  };

  auto attend = [&](int s, int slot) {
    const int kb = 64 * s;
    floatx16 x0, x1;
#pragma unroll
    for (int r = 0; r < 16; ++r) x0[r] = x1[r] = 0.f;
    {
      const uint8_t *lk = ldsk + (4 * slot + (kn >> 4)) * TB + (kn & 15) * 16;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        bf16x8 a0, a1;
        if constexpr (FP8) {
          const u32x2 w0 = *reinterpret_cast<const u32x2 *>(lk + j * 256 + 8 * hh);
          const u32x2 w1 = *reinterpret_cast<const u32x2 *>(lk + 2 * TB + j * 256 + 8 * hh);
          a0 = fp8x8_to_bf16x8(w0[0], w0[1]);
          a1 = fp8x8_to_bf16x8(w1[0], w1[1]);
        } else {
          a0 = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(lk + (2 * j + hh) * 256));
          a1 = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(lk + 2 * TB + (2 * j + hh) * 256));
        }
        x0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a0, qb[j], x0, 0, 0, 0);
        x1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a1, qb[j], x1, 0, 0, 0);
      }
    }
    const u32x4 okw = *reinterpret_cast<const u32x4 *>(s_ok[slot]);
    float mul[4], vsc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      mul[t] = FP8 ? a.scale_log2 * s_ks[slot][t] : a.scale_log2;
      vsc[t] = FP8 ? s_vs[slot][t] : 1.f;
    }
    // exponents against the reference maximum
    const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x0[r] = __builtin_fmaf(x0[r], mul[r >> 3], -m_use);
      x1[r] = __builtin_fmaf(x1[r], mul[2 + (r >> 3)], -m_use);
    }
    const uint32_t ok = __builtin_amdgcn_readfirstlane(okw[0] | okw[1] << 1 | okw[2] << 2 | okw[3] << 3);
    const bool masked = ok != 15u || kb + 64 > ctx;  // uniform
    uint64_t seen = ~0ull;                           // key kb + i is seen by this lane's row
    if (masked) {
      const int first = kb - ctx;  // the node of the step's first key
      if (first <= -64) {
      } else if (first < 0) {
        seen = ((1ull << -first) - 1ull) | (s_mask[32 * wave + n][0] << -first);
      } else {
        const int w = first >> 6, sh = first & 63;
        const uint64_t lo = w < WKV_TREE_MAX_WORDS ? s_mask[32 * wave + n][w & 3] : 0ull;
        const uint64_t hi = w + 1 < WKV_TREE_MAX_WORDS ? s_mask[32 * wave + n][(w + 1) & 3] : 0ull;
        seen = sh ? (lo >> sh) | (hi << (64 - sh)) : lo;
      }
      const int left = L - kb;
      if (left < 64) seen &= (1ull << left) - 1ull;
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (!(ok >> t & 1)) seen &= ~(0xFFFFull << (16 * t));
      const uint64_t v = seen >> (8 * hh);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if (!(v >> (16 * (r >> 3) + (r & 7)) & 1)) x0[r] = -INFINITY;
        if (!(v >> (32 + 16 * (r >> 3) + (r & 7)) & 1)) x1[r] = -INFINITY;
      }
    }
    float mt0 = fmaxf(x0[0], x0[1]), mt1 = fmaxf(x1[0], x1[1]);
#pragma unroll
    for (int r = 2; r < 16; r += 2) {
      mt0 = fmaxf(fmaxf(mt0, x0[r]), x0[r + 1]);
      mt1 = fmaxf(fmaxf(mt1, x1[r]), x1[r + 1]);
    }
    float mt = fmaxf(mt0, mt1);
    {
      const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
      mt = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
    }
    const bool unset = m_ref == -INFINITY;
    const bool move = unset ? mt > -INFINITY : mt > SOFTMAX_TAU;
    if (__any(move)) {  // rare after the first step
      const float sh = move ? mt : 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        x0[r] -= sh;
        x1[r] -= sh;
      }
      const float corr = move && !unset ? fast_exp2(-sh) : 1.f;
      l_part *= corr;
      if (move) m_ref = m_use + sh;
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[c][r] *= corr;
    }
    // probabilities, their sum and the PV operands
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x0[r] = fast_exp2(x0[r]);
      x1[r] = fast_exp2(x1[r]);
    }
    uint32_t pw[4][4];
    float ps = 0.f;
    if constexpr (FP8) {
      float p0 = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        ps += x0[r];
        p0 += x1[r];
      }
      ps += p0;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const floatx16 &sv = t < 2 ? x0 : x1;
      const int e0 = 8 * (t & 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (FP8) {
          pw[t][i] = pack_bf16x2(sv[e0 + 2 * i] * vsc[t], sv[e0 + 2 * i + 1] * vsc[t]);
        } else {  // the sum of the rounded probabilities that the products take
          pw[t][i] = pack_bf16x2(sv[e0 + 2 * i], sv[e0 + 2 * i + 1]);
          ps = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pw[t][i]), ones, ps, false);
        }
      }
    }
    l_part += ps;
    if (!masked) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const bf16x8 pb = __builtin_bit_cast(bf16x8, (u32x4{pw[t][0], pw[t][1], pw[t][2], pw[t][3]}));
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
          o[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v_operand(slot, t, c)), pb, o[c], 0,
                                                         0, 0);
      }
      return;
    }
#pragma unroll 1
    for (int t = 0; t < 4; ++t) {
      const int left = L - kb - 16 * t;
      if (left <= 0 || !(ok >> t & 1)) continue;  // uniform
      u32x4 pt = t == 0   ? u32x4{pw[0][0], pw[0][1], pw[0][2], pw[0][3]}
                 : t == 1 ? u32x4{pw[1][0], pw[1][1], pw[1][2], pw[1][3]}
                 : t == 2 ? u32x4{pw[2][0], pw[2][1], pw[2][2], pw[2][3]}
                          : u32x4{pw[3][0], pw[3][1], pw[3][2], pw[3][3]};
      // slots past the last token may hold anything: zeros in their place
      u32x4 real;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        real[i] = (8 * hh + 2 * i < left ? 0xFFFFu : 0u) | (8 * hh + 2 * i + 1 < left ? 0xFFFF0000u : 0u);
      u32x4 w[D / 32];
      bool odd = false;  // a V that is not finite
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        w[c] = v_operand(slot, t, c) & real;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          odd = odd || (w[c][i] & 0x7F80u) == 0x7F80u || (w[c][i] & 0x7F800000u) == 0x7F800000u;
      }
      if (!__any(odd)) {
        const bf16x8 pb = __builtin_bit_cast(bf16x8, pt);
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
          o[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, w[c]), pb, o[c], 0, 0, 0);
      } else {
#pragma unroll 1
        for (int e = 0; e < 16 && e < left; ++e) {
          const uint32_t word = (e & 7) < 2 ? pt[0] : (e & 7) < 4 ? pt[1] : (e & 7) < 6 ? pt[2] : pt[3];
          const uint32_t got = __shfl(word, n + 32 * (e >> 3), 64);
          const float p = bf16_bits_to_f32((e & 1) ? got >> 16 : got & 0xFFFFu);
          if (seen >> (16 * t + e) & 1) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
#pragma unroll
              for (int r = 0; r < 16; ++r)
                o[c][r] = __builtin_fmaf(p, v_value(slot, t, 32 * c + 8 * (r >> 2) + 4 * hh + (r & 3), e), o[c][r]);
              __builtin_amdgcn_sched_barrier(0);  // (few loads at a time: this path must not cost the others registers)
            }
          }
        }
      }
    }
  };

#pragma unroll
  for (int i = 0; i < NS - 1; ++i) issue(s0 + i, i);
  int slot = 0;
  for (int s = s0; s < s1; ++s) {
    wait_step();    // this wave's tile of step s
    barrier_lds();  // every wave's; every wave is done with step s - 1, whose slot takes step s + NS - 1
    const int next = slot == 0 ? NS - 1 : slot - 1;
    issue(s + NS - 1, next);
    if (active) attend(s, slot);
    slot = slot + 1 == NS ? 0 : slot + 1;
  }
  if (!active) return;
  float l = l_part;
  {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  if (tc.n > 1) {  // uniform
    float *pp = a.part + ((static_cast<int64_t>(b * a.Hkv + kvh) * a.units + unit) * a.chunks + chunk) * tree_part_floats<D>();
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<floatx4 *>(pp + ((4 * c + g) * 64 + lane) * 4) =
            floatx4{o[c][4 * g], o[c][4 * g + 1], o[c][4 * g + 2], o[c][4 * g + 3]};
    if (hh == 0) {
      pp[32 * D + n] = m_ref;
      pp[32 * D + 32 + n] = l;
    }
  } else if (has_row) {
    const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
    if (a.sinks != nullptr) l += exp2f(a.sinks[h] * 1.4426950408889634f - m_use);
    const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g)  // d = 32 c + 8 g + 4 hh + 0..3
        *reinterpret_cast<u32x2 *>(op + 32 * c + 8 * g + 4 * hh) =
            u32x2{pack_bf16x2(o[c][4 * g] * inv, o[c][4 * g + 1] * inv),
                  pack_bf16x2(o[c][4 * g + 2] * inv, o[c][4 * g + 3] * inv)};
  }
}

// Log-sum-exp merge of a unit's chunks: one wave per unit and 32 output columns.
// A sequence of one chunk was finished by the attention kernel.
template <int D>
__global__ __launch_bounds__(64) void tree_merge_kernel(TreeArgs a) {
  constexpr int PF = tree_part_floats<D>();
  const int lane = threadIdx.x, n = lane & 31, hh = lane >> 5;
  const int unit = blockIdx.x, c = blockIdx.z;
  const int kvh = blockIdx.y % a.Hkv, b = blockIdx.y / a.Hkv;
  const int q0 = a.cu_q[b], qlen = a.cu_q[b + 1] - q0;
  int L = a.seq_lens[b];
  L = L < a.max_seq ? L : a.max_seq;
  const int rows = qlen * a.G;
  if (qlen <= 0 || L <= 0 || 32 * unit >= rows) return;
  const int chunks = tree_chunks(L, a.chunk_steps, (L + 63) >> 6).n;
  if (chunks <= 1) return;
  const float *p = a.part + (static_cast<int64_t>(b * a.Hkv + kvh) * a.units + unit) * a.chunks * PF;
  float M = -INFINITY;
#pragma unroll 4
  for (int i = 0; i < chunks; ++i) M = fmaxf(M, p[i * static_cast<int64_t>(PF) + 32 * D + n]);
  const int row = 32 * unit + n;
  const bool has_row = row < rows;
  const int node = has_row ? row / a.by_G : 0, h = kvh * a.G + (has_row ? row - node * a.G : 0);
  const float m_use = M == -INFINITY ? 0.f : M;
  float l = 0.f;
  floatx4 acc[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) acc[g] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = 0; i < chunks; ++i) {
    const float *ps = p + i * static_cast<int64_t>(PF);
    const float w = exp2f(ps[32 * D + n] - m_use);  // 0 for a chunk of which the row saw no key
    l += w * ps[32 * D + 32 + n];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const floatx4 x = *reinterpret_cast<const floatx4 *>(ps + ((4 * c + g) * 64 + lane) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[g][e] += w * x[e];
    }
  }
  if (!has_row) return;
  if (a.sinks != nullptr) l += exp2f(a.sinks[h] * 1.4426950408889634f - m_use);
  const float inv = l != 0.f ? 1.f / l : 0.f;
  uint16_t *op = a.out + static_cast<int64_t>(q0 + node) * a.o_st + static_cast<int64_t>(h) * a.o_sh;
#pragma unroll
  for (int g = 0; g < 4; ++g)
    *reinterpret_cast<u32x2 *>(op + 32 * c + 8 * g + 4 * hh) =
        u32x2{pack_bf16x2(acc[g][0] * inv, acc[g][1] * inv), pack_bf16x2(acc[g][2] * inv, acc[g][3] * inv)};
}

// How a launch covers its work.
struct TreePlan {
  int units;        // per (sequence, KV head) at the longest query
  int row_groups;   // workgroups of them
  int chunks, chunk_steps;
};

// Chunks: enough workgroups for two per CU, of at least four steps each.
static TreePlan tree_plan(int batch, int Hkv, int G, int max_query_len, int max_seq, bool cut) {
  TreePlan p;
  p.units = static_cast<int>((static_cast<int64_t>(max_query_len) * G + 31) / 32);
  p.row_groups = (p.units + kTreeWaves - 1) / kTreeWaves;
  const int steps = (max_seq + 63) / 64;
  const int64_t wgs = static_cast<int64_t>(batch) * Hkv * p.row_groups;
  int64_t chunks = cut ? (2 * kTreeCus + wgs - 1) / wgs : 1;
  const int most = steps / 4 > 1 ? steps / 4 : 1;
  if (chunks > most) chunks = most;
  p.chunk_steps = static_cast<int>((steps + chunks - 1) / chunks);
  if (p.chunk_steps < 1) p.chunk_steps = 1;
  p.chunks = steps > 0 ? (steps + p.chunk_steps - 1) / p.chunk_steps : 1;
  return p;
}

static int64_t tree_workspace(const TreePlan &p, int batch, int Hkv, int D) {
  return p.chunks > 1 ? static_cast<int64_t>(batch) * Hkv * p.units * p.chunks * (32 * D + 64) * 4 : 0;
}

}  // namespace wkv

using namespace wkv;

extern "C" int64_t wkv_tree_workspace_size(int32_t batch, int32_t kv_dtype, int32_t num_kv_heads, int32_t num_q_heads,
                                           int32_t head_dim, int32_t max_query_len, int32_t max_seq_len) {
  if (batch < 0 || batch > 65535 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads != 0 ||
      (head_dim != 64 && head_dim != 128) || max_query_len < 0 || max_seq_len < 0 ||
      (kv_dtype != WKV_KV_BF16 && kv_dtype != WKV_KV_FP8_E4M3) ||
      static_cast<int64_t>(max_query_len) * (num_q_heads / num_kv_heads) > (1 << 24))
    return -1;
  if (batch == 0 || max_query_len == 0) return 0;
  const TreePlan p = tree_plan(batch, num_kv_heads, num_q_heads / num_kv_heads, max_query_len, max_seq_len, true);
  return tree_workspace(p, batch, num_kv_heads, head_dim);
}

extern "C" int wkv_tree_gqa(const wkv_cache_t *cache, const void *key, int64_t key_stride_t, int64_t key_stride_h,
                            const void *value, int64_t value_stride_t, int64_t value_stride_h,
                            const int64_t *slot_mapping, int64_t num_tokens, const void *q, int64_t q_stride_t,
                            int64_t q_stride_h, void *out, int64_t out_stride_t, int64_t out_stride_h,
                            int32_t num_q_heads, const int32_t *cu_seqlens_q, const int32_t *seq_lens,
                            const int32_t *block_table, int64_t bt_stride, int32_t max_blocks_per_seq, int32_t batch,
                            int32_t max_query_len, int32_t max_seq_len, const int64_t *tree_mask, int32_t mask_words,
                            float scale, void *workspace, int64_t workspace_bytes, const float *sinks, void *stream) {
  int rc = check_cache(cache, -1);
  if (rc) return rc;
  WKV_CHECK_ARG(batch >= 0 && batch <= 65535, "batch must be in [0, 65535] (got %d)", batch);
  WKV_CHECK_ARG(num_tokens >= 0, "num_tokens must be >= 0");
  // The drafted tokens go into the cache first (same stream), once nothing is left to refuse.
  auto append = [&]() -> int {
    if (key == nullptr && value == nullptr && slot_mapping == nullptr) return WKV_OK;
    return cache->kv_dtype == WKV_KV_FP8_E4M3
               ? wkv_append_fp8(cache, key, key_stride_t, key_stride_h, value, value_stride_t, value_stride_h,
                                slot_mapping, num_tokens, stream)
               : wkv_append(cache, key, key_stride_t, key_stride_h, value, value_stride_t, value_stride_h,
                            slot_mapping, num_tokens, stream);
  };
  if (batch == 0 || max_query_len == 0) return append();
  const int Hkv = cache->num_kv_heads, D = cache->head_dim, BS = cache->block_size;
  WKV_CHECK_ARG(num_q_heads > 0 && num_q_heads % Hkv == 0, "num_q_heads %d must be a multiple of num_kv_heads %d",
                num_q_heads, Hkv);
  const int G = num_q_heads / Hkv;
  WKV_CHECK_ARG(cache->num_blocks * Hkv <= INT32_MAX, "num_blocks * num_kv_heads must be below 2^31");
  WKV_CHECK_ARG(q != nullptr && aligned16(q), "q must be non-NULL and 16-byte aligned");
  WKV_CHECK_ARG(q_stride_t >= 0 && q_stride_h >= 0 && q_stride_t % 8 == 0 && q_stride_h % 8 == 0,
                "q strides must be non-negative multiples of 8");
  WKV_CHECK_ARG(out != nullptr && aligned16(out), "out must be non-NULL and 16-byte aligned");
  WKV_CHECK_ARG(out_stride_t >= 0 && out_stride_h >= 0 && out_stride_t % 4 == 0 && out_stride_h % 4 == 0,
                "out strides must be non-negative multiples of 4");
  WKV_CHECK_ARG(cu_seqlens_q != nullptr && seq_lens != nullptr && block_table != nullptr,
                "cu_seqlens_q / seq_lens / block_table is NULL");
  WKV_CHECK_ARG(max_blocks_per_seq > 0 && bt_stride >= max_blocks_per_seq, "bad block table geometry");
  WKV_CHECK_ARG(max_query_len > 0 && max_seq_len >= 0, "max_query_len must be > 0 and max_seq_len >= 0");
  WKV_CHECK_ARG(tree_mask != nullptr && reinterpret_cast<uintptr_t>(tree_mask) % 8 == 0, "tree_mask must be non-NULL int64");
  WKV_CHECK_ARG(mask_words >= 1 && mask_words <= WKV_TREE_MAX_WORDS, "mask_words must be in [1, %d] (got %d)",
                WKV_TREE_MAX_WORDS, mask_words);
  WKV_CHECK_ARG(std::isfinite(scale), "scale must be finite");
  WKV_CHECK_ARG(reinterpret_cast<uintptr_t>(sinks) % 4 == 0, "sinks must be fp32");
  WKV_CHECK_ARG(static_cast<int64_t>(max_query_len) * G <= (1 << 24), "max_query_len * query heads per KV head too large");
  const int64_t table_tokens = static_cast<int64_t>(max_blocks_per_seq) * BS;
  const int max_seq = max_seq_len < table_tokens ? max_seq_len : static_cast<int>(table_tokens);
  const TreePlan p = tree_plan(batch, Hkv, G, max_query_len, max_seq, workspace != nullptr);
  const int64_t need = tree_workspace(p, batch, Hkv, D);
  if (need > 0)
    WKV_CHECK_ARG(aligned16(workspace) && workspace_bytes >= need, "workspace too small: need %lld bytes, got %lld",
                  (long long)need, (long long)workspace_bytes);
  const int64_t items = static_cast<int64_t>(batch) * p.chunks * Hkv;
  WKV_CHECK_ARG(items <= 8 * 65535 && static_cast<int64_t>(batch) * Hkv <= 65535, "too many sequences and KV heads");
  rc = append();
  if (rc) return rc;
  const TreeArgs a{static_cast<const uint8_t *>(cache->k), static_cast<const uint8_t *>(cache->v), cache->k_scale,
                   cache->v_scale, static_cast<const uint16_t *>(q), q_stride_t, q_stride_h,
                   static_cast<uint16_t *>(out), out_stride_t, out_stride_h, cu_seqlens_q, seq_lens, block_table,
                   bt_stride, tree_mask, mask_words, max_blocks_per_seq, max_seq, Hkv, G, BS,
                   static_cast<int>(cache->num_blocks), fast_div(BS), fast_div(G), fast_div(Hkv), fast_div(p.chunks),
                   static_cast<int>(items), p.chunks, p.chunk_steps, p.units, scale * 1.4426950408889634f,
                   static_cast<float *>(workspace), sinks};
  const dim3 grid(static_cast<unsigned>(8 * p.row_groups), static_cast<unsigned>((items + 7) / 8));
  auto s = static_cast<hipStream_t>(stream);
  const bool fp8 = cache->kv_dtype == WKV_KV_FP8_E4M3;
#define WKV_TREE(Dv, F8) tree_gqa_kernel<Dv, F8, tree_steps_in_lds<Dv, F8>()><<<grid, 64 * kTreeWaves, 0, s>>>(a)
  if (D == 128) {
    if (fp8) WKV_TREE(128, true); else WKV_TREE(128, false);
  } else {
    if (fp8) WKV_TREE(64, true); else WKV_TREE(64, false);
  }
#undef WKV_TREE
  WKV_CHECK_LAUNCH("tree attention");
  if (p.chunks > 1) {
    const dim3 mgrid(static_cast<unsigned>(p.units), static_cast<unsigned>(batch * Hkv), static_cast<unsigned>(D / 32));
    if (D == 128)
      tree_merge_kernel<128><<<mgrid, 64, 0, s>>>(a);
    else
      tree_merge_kernel<64><<<mgrid, 64, 0, s>>>(a);
    WKV_CHECK_LAUNCH("tree attention merge");
  }
  return WKV_OK;
}
