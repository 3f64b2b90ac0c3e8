// The accepted path's keys and values moved together (gfx950): of every
// sequence, the tokens at positions seq_lens + path[0 .. accepted) to positions
// seq_lens + 0, 1, .. in the paged cache, in place. A rising path names no node
// before its place (path[j] >= j), so the tokens that keep their place lead and
// only those behind them are touched.
//
// One workgroup per (sequence, KV head): every moved token's K and V row is
// read into LDS before anything is written (a token's new place can be another's
// old one), as bf16 values. bf16 caches copy 16-byte K chunks and single V elements (a token's
// V lies across the block's rows). fp8 caches decode exactly, then append each
// new block's tokens as one run, with the append kernel's own run (one wave a
// run): the block's earlier codes are encoded again where its scale grows.
// Bound by two round trips to memory and the launch: the bytes of a step (64
// sequences x 8 tokens x 8 heads) are 4 MB. That step in bf16 5.2 us; 33 sequences x up
// to 12 tokens x 4 heads in fp8 10.0 us, half of it the runs of the append rule: a run is one wave's
// chain of loads, maximum, scale and codes, and a path that fits one block is one run.
//
// fp8 costs accuracy that a bf16 cache does not: a moved token has been rounded twice (to
// half a step of e4m3, 2^-4 of it, each time), and a block keeps the scale of the largest token that was
// drafted into it, rejected ones too, until it is begun afresh -- as the append rule has it.
#include "kv_append_dev.h"

namespace wkv {

constexpr int kCompactWaves = 4;

template <int D, bool FP8>
__global__ __launch_bounds__(64 * kCompactWaves) void compact_kernel(
    uint8_t *kc, uint8_t *vc, float *ks, float *vs, const int32_t *__restrict__ bt, int64_t bt_stride, int Mb,
    const int32_t *__restrict__ seq_lens, const int32_t *__restrict__ path, int path_len,
    const int32_t *__restrict__ accepted, int H, int BS, int64_t NB) {
  constexpr int P = WKV_TREE_MAX_DEPTH;
  constexpr int KP = D + 8;  // LDS row of a token, in elements: 16-byte steps, the rows on different banks
  __shared__ __attribute__((aligned(16))) uint16_t rk[P * KP], rv[P * KP];
  struct Place {
    int blk, off;  // block (-1: none) and offset in it
  };
  __shared__ Place src[P], dst[P];  // of the moved tokens that have both
  __shared__ int64_t slots[P];      // of the new places, for the fp8 runs
  __shared__ int moved;
  const int b = blockIdx.y, h = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int L = max(seq_lens[b], 0);
  int n = accepted[b];
  n = n < path_len ? n : path_len;
  // Every wave finds the moved tokens by itself: lane j holds path entry j.
  const int mine = lane < n ? path[static_cast<int64_t>(b) * path_len + lane] : lane;
  const uint64_t off = __ballot(mine != lane);
  if (off == 0) return;  // the whole workgroup
  const int j0 = __builtin_ctzll(off);  // path entries j0 .. n - 1 move
  const int32_t *row = bt + b * bt_stride;
  auto place = [&](int64_t pos) {
    if (pos < 0 || pos >= static_cast<int64_t>(Mb) * BS || pos > INT32_MAX) return Place{-1, 0};
    const int i = static_cast<int>(pos) / BS, blk = row[i];
    return blk >= 0 && blk < NB ? Place{blk, static_cast<int>(pos) - i * BS} : Place{-1, 0};
  };
  if (wave == 0) {  // uniform. What has no place before or after is left out, so that a block's tokens are one run.
    Place d{-1, 0}, s{-1, 0};
    if (lane >= j0 && lane < n && mine != lane) {
      d = place(static_cast<int64_t>(L) + lane);
      if (mine >= 0) s = place(static_cast<int64_t>(L) + mine);
    }
    const bool both = d.blk >= 0 && s.blk >= 0;
    const uint64_t kept = __ballot(both);
    if (both) {
      const int t = __builtin_popcountll(kept & ((1ull << lane) - 1ull));
      src[t] = s;
      dst[t] = d;
      slots[t] = static_cast<int64_t>(d.blk) * BS + d.off;
    }
    if (lane == 0) moved = __builtin_popcountll(kept);
  }
  auto region = [&](const Place &x) { return static_cast<int64_t>(x.blk) * H + h; };
  __syncthreads();
  const int m = __builtin_amdgcn_readfirstlane(moved);
  constexpr int X = FP8 ? 16 : 8;  // elements of a K chunk
  constexpr int NC = D / X;
  for (int i = tid; i < m * NC; i += 64 * kCompactWaves) {
    const int t = i / NC, c = i % NC;
    const Place s = src[t];
    const u32x4 w = *reinterpret_cast<const u32x4 *>(kc + ((region(s) * NC + c) * BS + s.off) * 16);
    if constexpr (FP8) {
      const float sc = ks[region(s)];
      u32x4 o[2];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float lo = e4m3_decode((w[e >> 1] >> (16 * (e & 1))) & 0xffu) * sc;
        const float hi = e4m3_decode((w[e >> 1] >> (16 * (e & 1) + 8)) & 0xffu) * sc;
        o[e >> 2][e & 3] = f32_to_bf16_bits(lo) | (f32_to_bf16_bits(hi) << 16);  // exact: a code has 4 significant bits
      }
      *reinterpret_cast<u32x4 *>(rk + t * KP + 16 * c) = o[0];
      *reinterpret_cast<u32x4 *>(rk + t * KP + 16 * c + 8) = o[1];
    } else {
      *reinterpret_cast<u32x4 *>(rk + t * KP + 8 * c) = w;
    }
  }
#pragma unroll 4
  for (int i = tid; i < m * D; i += 64 * kCompactWaves) {
    const int t = i / D, d = i % D;
    const Place s = src[t];
    const int64_t at = (region(s) * D + d) * BS + s.off;
    if constexpr (FP8)
      rv[t * KP + d] = static_cast<uint16_t>(f32_to_bf16_bits(e4m3_decode(vc[at]) * vs[region(s)]));
    else
      rv[t * KP + d] = reinterpret_cast<const uint16_t *>(vc)[at];
  }
  __syncthreads();
  if constexpr (!FP8) {
    for (int i = tid; i < m * NC; i += 64 * kCompactWaves) {
      const int t = i / NC, c = i % NC;
      const Place s = dst[t];
      *reinterpret_cast<u32x4 *>(kc + ((region(s) * NC + c) * BS + s.off) * 16) =
          *reinterpret_cast<const u32x4 *>(rk + t * KP + 8 * c);
    }
#pragma unroll 4
    for (int i = tid; i < m * D; i += 64 * kCompactWaves) {
      const int t = i / D, d = i % D;
      const Place s = dst[t];
      reinterpret_cast<uint16_t *>(vc)[(region(s) * D + d) * BS + s.off] = rv[t * KP + d];
    }
  } else {
    // Runs: the new places by block, in turn over the waves -- one run a block, as two waves
    // at one block would race.
    int run = 0;
    for (int t = 0; t < m;) {  // uniform
      const int blk = __builtin_amdgcn_readfirstlane(dst[t].blk), first = __builtin_amdgcn_readfirstlane(dst[t].off);
      int r = 1;
      while (t + r < m && dst[t + r].blk == blk) ++r;
      r = __builtin_amdgcn_readfirstlane(r);
      if (run % kCompactWaves == wave)
        fp8_append_run_kv<D>(kc, vc, ks, vs, rk, KP, 0, rv, KP, 0, slots, t, r, blk, first, h, H, BS);
      ++run;
      t += r;
    }
  }
}

}  // namespace wkv

using namespace wkv;

extern "C" int wkv_compact(const wkv_cache_t *cache, const int32_t *block_table, int64_t bt_stride,
                           int32_t max_blocks_per_seq, const int32_t *seq_lens, const int32_t *path, int32_t path_len,
                           const int32_t *accepted, int32_t batch, void *stream) {
  int rc = check_cache(cache, -1);
  if (rc) return rc;
  WKV_CHECK_ARG(batch >= 0 && batch <= 65535, "batch must be in [0, 65535] (got %d)", batch);
  WKV_CHECK_ARG(path_len > 0 && path_len <= WKV_TREE_MAX_DEPTH, "path_len must be in [1, %d] (got %d)",
                WKV_TREE_MAX_DEPTH, path_len);
  if (batch == 0) return WKV_OK;
  WKV_CHECK_ARG(block_table != nullptr && seq_lens != nullptr && path != nullptr && accepted != nullptr,
                "block_table / seq_lens / path / accepted is NULL");
  WKV_CHECK_ARG(max_blocks_per_seq > 0 && bt_stride >= max_blocks_per_seq, "bad block table geometry");
  const dim3 grid(static_cast<unsigned>(cache->num_kv_heads), static_cast<unsigned>(batch));
  auto s = static_cast<hipStream_t>(stream);
  auto kc = static_cast<uint8_t *>(cache->k), vc = static_cast<uint8_t *>(cache->v);
#define WKV_COMPACT(Dv, F8)                                                                                        \
  compact_kernel<Dv, F8><<<grid, 64 * kCompactWaves, 0, s>>>(kc, vc, cache->k_scale, cache->v_scale, block_table,  \
                                                             bt_stride, max_blocks_per_seq, seq_lens, path,        \
                                                             path_len, accepted, cache->num_kv_heads,              \
                                                             cache->block_size, cache->num_blocks)
  const bool fp8 = cache->kv_dtype == WKV_KV_FP8_E4M3;
  if (cache->head_dim == 128) {
    if (fp8) WKV_COMPACT(128, true); else WKV_COMPACT(128, false);
  } else {
    if (fp8) WKV_COMPACT(64, true); else WKV_COMPACT(64, false);
  }
#undef WKV_COMPACT
  WKV_CHECK_LAUNCH("compact");
  return WKV_OK;
}
