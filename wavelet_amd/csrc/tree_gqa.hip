// Attention of a tree of drafted tokens over the paged cache (gfx950).
//
// Sequence b brings n_b drafted tokens (the last n_b of its L_b = seq_lens[b])
// and every one of its G query heads per KV head: n_b G rows of one KV head that
// read the same keys. All rows see the context's keys; of the drafted tokens'
// keys a row sees those whose bit its mask sets.
//
// Work: the rows of one (sequence, KV head), node by node with the G heads of a
// node together, are taken 32 at a time by a wave (a unit: the columns of its
// 32x32x16 MFMAs), four units to a workgroup (a row group), so that up to 128
// rows share one read of the keys. Keys go in steps of 64, copied to LDS by
// LDS-DMA, a 16-key tile by each wave. A row group of at most two units has two waves
// on each, for 32 keys of every step each, and joins them in LDS; in a larger one a
// wave without rows only copies. The
// steps of all row groups form one line that the workgroups share evenly
// (tree_prefix), whatever the mix of lengths; a row group cut between workgroups
// leaves fp32 partials that a second kernel merges by log-sum-exp. Row groups enough for the
// chip and of like lengths stay whole instead, one to a workgroup (tree_whole).
//
// Bound by reading K and V once for up to 64 rows of bf16, by the step's own chain
// (products, exponents, the copies' issue, a barrier) past that and in fp8. Measured, 32 query and
// 8 KV heads of 128, with the drafted tokens' append: 64 sequences of 4,096 tokens with 16 drafted
// each, bf16, 184 us (6.0 TB/s; a chunk of each sequence per workgroup, with cached reads: 206); 6 of
// 3,000 to 24,000 with 5 to 63 drafted, 28 and 4 heads, fp8, 67 to 72 us (400 TFLOP/s;
// chunks: 172); 64 of 4,096 with 8 drafted, fp8, 120 us (4.5 TB/s; with one wave per unit
// 137); 4 of 8,192 with 128 drafted 111 to 115 us in bf16 and 106 to 112 in fp8 (610 and 640 TFLOP/s; the
// matrix unit is busy 41% of the time, the VALU 38%). Chunks took 111 and 108 there: even shares
// gain nothing where the sequences are alike and wide.
//
// Software pipeline, one barrier per step: while a wave finishes step s
// (probabilities, PV products) it scores step s + 1, so that the matrix unit
// and the VALU work at the same time. At the barrier of step s every wave's V of
// step s and K of step s + 1 have landed; their slots before (two each) take V of
// step s + 1 and K of step s + 2. fp8 tiles land as codes in their bf16 tile's place and
// are widened there, at their block's scale (exact), by the wave that copied them.
//
// Rounding: scores, exponents, maxima, sums, outputs in progress and partials are fp32. Probabilities
// are rounded to bf16 for the PV product, as the prompt kernel has them (the bf16 MFMA is the fast one;
// the sum is of the rounded ones, so that a row of equal values keeps them): each is off
// by at most 2^-9 of itself, independently, which is an error the size of the bf16 output's own
// rounding -- together sqrt(2) of it, 2.3e-3 of the result's norm against 1.7e-3 with fp32 probabilities.
//
// Masked keys: scores are set to -inf after scaling (a step's window of the row's
// mask, 64 bits), so that neither the scale's sign nor a NaN key matters. A masked
// probability is 0, but 0 times a V that is not finite is NaN: in steps that
// mask anything, such a V goes apart, to the rows that see its key.
#include <cmath>
#include <type_traits>

#include "gqa_tiles.h"
#include "lds_dma.h"

namespace wkv {

typedef __attribute__((__vector_size__(2 * sizeof(uint16_t)))) uint16_t u16x2;

constexpr int kTreeWaves = 4;
constexpr int kTreeRows = 32 * kTreeWaves;  // rows of a workgroup
constexpr int kTreeShare = 512;  // workgroups that share a launch's steps: two per CU
constexpr int kTreeMost = 2048;  // of a launch that may share them or have one per row group

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
  int batch, Mb, max_seq, Hkv, G, BS, nb;
  FastDiv by_BS, by_G;
  int share;   // workgroups that may share the line; 0: one per row group
  int groups;  // row groups per (sequence, KV head) at the longest query
  int stream;  // blocks are read by one sequence
  float scale_log2;
  float *part;
  const float *sinks;
};

// The kernel's arguments, read again from the kernel-argument segment (the
// pointer is opaque to the compiler): held across the loop over row groups they
// would spill scalar registers into the key loop.
__device__ __forceinline__ const TreeArgs &tree_args() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const TreeArgs *)(p);
}

// A sequence's share of the line, per KV head: `groups` row groups of `steps` steps each
// (a sequence without keys counts one: its rows are written all the same). The drafted tokens are
// the last of all its tokens; of those past max_seq no key is read.
struct TreeSeq {
  int qlen, ctx, L, steps, groups;  // rows, cached tokens, tokens that are read
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs &a, int b) {
  TreeSeq s;
  s.qlen = a.cu_q[b + 1] - a.cu_q[b];
  s.L = a.seq_lens[b];
  s.ctx = s.L - s.qlen;
  s.L = s.L < a.max_seq ? s.L : a.max_seq;
  s.steps = s.L > 0 ? (s.L + 63) >> 6 : 1;
  s.groups = s.qlen > 0 ? (s.qlen * a.G + kTreeRows - 1) / kTreeRows : 0;
  return s;
}

// The line: KV head by KV head, sequence by sequence, row group by row group,
// step by step. Every workgroup forms its prefix itself: each thread adds up a
// run of `per` sequences; pfx[t] (LDS) is the sum before thread t's run, of steps, and
// pfx[kTreeThreads + t] of row groups.
constexpr int kTreeThreads = 64 * kTreeWaves;
struct TreeLine {
  int steps, groups, longest;  // of one KV head; steps of the longest sequence
};
__device__ __forceinline__ TreeLine tree_prefix(const TreeArgs &a, int *pfx, int per) {
  int steps = 0, groups = 0, longest = 0;
  for (int b = threadIdx.x * per; b < a.batch && b < static_cast<int>(threadIdx.x + 1) * per; ++b) {
    const TreeSeq s = tree_seq(a, b);
    steps += s.steps * s.groups;
    groups += s.groups;
    if (s.groups > 0) longest = max(longest, s.steps);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int *const red = pfx + 2 * kTreeThreads;
  int sum = steps, sum_g = groups;  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(sum, o, 64), z = __shfl_up(sum_g, o, 64), m = __shfl_xor(longest, o, 64);
    if (lane >= o) {
      sum += y;
      sum_g += z;
    }
    longest = max(longest, m);
  }
  if (lane == 63) {
    red[wave] = sum;
    red[kTreeWaves + wave] = sum_g;
    red[2 * kTreeWaves + wave] = longest;
  }
  __syncthreads();
  int before = 0, before_g = 0;
  longest = 0;
#pragma unroll
  for (int w = 0; w < kTreeWaves; ++w) {
    if (w == wave) {
      pfx[threadIdx.x] = before + sum - steps;
      pfx[kTreeThreads + threadIdx.x] = before_g + sum_g - groups;
    }
    before += red[w];
    before_g += red[kTreeWaves + w];
    longest = max(longest, red[2 * kTreeWaves + w]);
  }
  __syncthreads();
  return TreeLine{__builtin_amdgcn_readfirstlane(before), __builtin_amdgcn_readfirstlane(before_g),
                  __builtin_amdgcn_readfirstlane(longest)};
}

// How many workgroups share a line of T steps: all of the grid, two per CU, with
// at least four steps each. bf16, 32 query and 8 KV heads of 128, us for 512 / 256 /
// 128 workgroups: eight shares' worth of steps each and more (sequences of 300 to
// 24,000 tokens) 68 / 85 / 125; 64 sequences of 600 to 2,000 tokens 41 / 46 / 62;
// one of 4,096 tokens (one step each / two / four) 32.5 / 26.7 / 26.8.
__device__ __forceinline__ int tree_workgroups(int T) {
  const int w = (T / 4) & ~7;
  return w < 8 ? 8 : (w < kTreeShare ? w : kTreeShare);
}

// Whether each of N row groups (T steps, the longest of `longest`) gets a workgroup of its
// own instead of even shares. Those cost the partials that cutting leaves and the merge reads,
// another start, and the meeting of row groups of the same keys in the L2; whole groups
// wait for the longest. By microseconds of a step alone on its CU, of one of two, and of a
// partial. Whole / shared, us (the one taken first):
//   32 and 8 heads of 128, bf16: 64 sequences of 700 to 1,000 tokens with 16 drafted 71 / 99, 128 of
//   100 to 1,000 with 8 to 32 105 / 130, 64 of 4,000 to 8,000 with 32 to 64 523 / 623; shared: 64
//   of 100 to 8,000 with 16 to 48 305 / 394;
//   the same heads, fp8: 64 of 700 to 1,000 43 / 69, 128 of 800 to 1,000 with 8 to 32 95 / 119; shared:
//   64 of 4,000 to 8,000 with 32 to 64 521 / 556, of 100 to 8,000 with 16 to 48 249 / 349;
//   14 and 2 heads of 64, bf16: 64 of 700 to 1,000 36 / 39, 128 of 1,000 to 1,400 with 8 to 32 50 / 56;
//   shared: 64 of 4,000 to 8,000 with 32 to 64 138 / 169, of 100 to 8,000 with 16 to 48 91 / 155 (fp8:
//   144 / 199 and 88 / 181).
template <int D, bool FP8>
__device__ __forceinline__ bool tree_whole(int T, int N, int longest, int items, int W) {
  constexpr float kAlone = 1.3f, kPair = 2.6f, kCut = D == 128 ? 60.f : 40.f, kPart = 0.026f * D / 128;
  const float line = static_cast<float>(T) / W * (W > kTreeShare / 2 ? kPair : kAlone);
  if (N <= kTreeShare / 2) return longest * kAlone <= line + 6.f + kPart * (W + N);
  const float mean = static_cast<float>(T) / N;
  const float again = FP8 || N <= items ? 0.f : 0.25f * line * (1.f - static_cast<float>(items) / N);
  return (longest - mean) * kAlone + 0.3f * mean <= kCut + again;
}

// The points of the line (steps, or whole row groups) over W workgroups: an even number each, one
// more for the first (W at most the points, below 2^31).
struct TreeShare {
  int each, more;
  __device__ __forceinline__ int begin(int w) const { return w * each + (w < more ? w : more); }
  __device__ __forceinline__ int of(int x) const {  // the workgroup of point x
    const int y = x - more * (each + 1);
    return y < 0 ? x / (each + 1) : more + y / each;
  }
};

// A unit's partial: D / 32 x 4 runs of 64 lanes x 4 fp32 (the output accumulators
// as the lanes hold them), then the 32 rows' reference maxima (log2 domain) and
// sums. Workgroup w owns slots 2 w (the row group that its share begins in) and
// 2 w + 1 (a later one), four units each. Behind them, per workgroup of the grid, in how many
// parts the row group is whose first one it left (0: none), and a record of it.
template <int D>
__host__ __device__ constexpr int tree_part_floats() {
  return 32 * D + 64;
}
struct TreeRec {
  int slot;  // of the first part
  int next;  // of the others, two apart: the first slots of the workgroups behind
  int b, kvh, group;
  int pad[3];
};
template <int D>
__device__ __forceinline__ int *tree_counts(float *part) {
  return reinterpret_cast<int *>(part + static_cast<int64_t>(kTreeShare) * 2 * kTreeWaves * tree_part_floats<D>());
}
template <int D>
__device__ __forceinline__ TreeRec *tree_records(float *part) {
  return reinterpret_cast<TreeRec *>(tree_counts<D>(part) + kTreeShare);
}

// Eight e4m3fn codes (bytes of lo, then hi) times a power-of-two scale as
// eight bf16 values (exact: every such product is a bf16 value).
__device__ __forceinline__ u32x4 codes_to_bf16(uint32_t lo, uint32_t hi, float sc) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, sc, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, sc, true)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, sc, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, sc, true))};
}

// The workgroups share the line (a.share of them), or take one row group each.
template <int D, bool FP8>
__global__ __launch_bounds__(kTreeThreads, 2) void tree_gqa_kernel(TreeArgs kernel_args) {
  constexpr int ESZ = FP8 ? 1 : 2;
  constexpr int TB = D * 16 * 2;           // bytes of a 16-key tile's K, and of its V, as bf16
  constexpr int NC = D * 16 * ESZ / 1024;  // 1 KB copies of each
  // bf16 tiles as the MFMAs read them: K [D / 8 chunks][16 tokens][16 bytes] as the
  // cache holds it, V [D rows][2 token octets][8 tokens] (the octets swapped in every second
  // eight rows). fp8 codes land at their tile's start: K [D / 16 chunks][16 tokens][16 bytes],
  // V [D rows][16 tokens].
  __shared__ __attribute__((aligned(16))) uint8_t ldsk[2 * 4 * TB];
  __shared__ __attribute__((aligned(16))) uint8_t ldsv[2 * 4 * TB];
  __shared__ __attribute__((aligned(16))) int s_ok[4][4];  // by step: the tile holds keys
  __shared__ TreeShare s_share;                            // how the line is shared, and
  __shared__ int s_place;                                  // this workgroup's place among those that do
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63, n = lane & 31, hh = lane >> 5;
  // The lane, for code off the hot path: what is formed from it stays there (hoisted
  // out of the key loop it would be spilled, and a reload waits for the copies in flight).
  auto lane_here = [&]() __attribute__((always_inline)) {
    int l = lane;
    asm volatile("" : "+v"(l));
    return l;
  };
  const int id = blockIdx.x;
  int b, kvh, rg, s_begin = 0;
  bool later = false;  // past the share's first row group
  int steps_left;      // of this workgroup's share
  if (kernel_args.share > 0) {
    const TreeArgs &a = tree_args();
    const int *pfx = reinterpret_cast<int *>(ldsk);
    const int per = (a.batch + kTreeThreads - 1) / kTreeThreads;
    const TreeLine line = tree_prefix(a, reinterpret_cast<int *>(ldsk), per);
    const int T = line.steps * a.Hkv, N = line.groups * a.Hkv;
    if (threadIdx.x == 0 && id < kTreeShare) tree_counts<D>(a.part)[id] = 0;
    // XCD i mod 8 takes a contiguous eighth of the line, whose workgroups read the same keys.
    int W = tree_workgroups(T);
    const bool whole = N <= static_cast<int>(gridDim.x) &&
                       tree_whole<D, FP8>(T, N, line.longest, a.batch * a.Hkv, W);  // uniform
    if (whole) W = (N + 7) & ~7;  // one each
    const int w = (id & 7) * (W / 8) + id / 8;
    if (id >= W) return;
    const int points = whole ? N : T;  // of the line
    W = points < W ? points : W;
    if (w >= W) return;
    TreeShare share;
    share.each = points / W;
    share.more = points - share.each * W;
    int y = share.begin(w);
    steps_left = share.begin(w + 1) - y;
    if (whole) pfx += kTreeThreads;
    const int head = whole ? line.groups : line.steps;
    kvh = y / head;
    y -= kvh * head;
    int lo = 0, hi = kTreeThreads;  // the last run that begins at or before y (empty runs share their successor's sum)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pfx[mid] <= y) lo = mid; else hi = mid;
    }
    y -= pfx[lo];
    for (b = lo * per;; ++b) {  // the run holds y
      const TreeSeq s = tree_seq(a, b);
      const int c = whole ? s.groups : s.steps * s.groups;
      if (y < c || b + 1 >= a.batch) {
        rg = whole ? y : y / s.steps;
        if (whole) steps_left = s.steps; else s_begin = y - rg * s.steps;
        break;
      }
      y -= c;
    }
    if (threadIdx.x == 0) {  // (read after the barriers of a row group)
      s_share = share;
      s_place = w;
    }
  } else {
    // The row groups of one item stand eight workgroups apart: on one XCD, whose
    // L2 then serves their keys.
    const TreeArgs &a = kernel_args;
    const int oct = id / (8 * a.groups), r = id - oct * 8 * a.groups;
    rg = r >> 3;
    const int item = 8 * oct + (r & 7);
    if (item >= a.batch * a.Hkv) return;
    b = item / a.Hkv;
    kvh = item - b * a.Hkv;
    const TreeSeq s = tree_seq(a, b);
    if (rg >= s.groups) return;
    // (the last one takes those past the longest query that the launch was told of, too: a sequence
    // that was refused for its many nodes has rows to clear)
    const int64_t all = static_cast<int64_t>(rg + 1 == a.groups ? s.groups - rg : 1) * s.steps;
    steps_left = all < INT32_MAX ? static_cast<int>(all) : INT32_MAX;
  }
  for (;;) {  // the row groups of the share
  const TreeArgs &a = tree_args();
  b = __builtin_amdgcn_readfirstlane(b);
  kvh = __builtin_amdgcn_readfirstlane(kvh);
  rg = __builtin_amdgcn_readfirstlane(rg);
  s_begin = __builtin_amdgcn_readfirstlane(s_begin);
  const TreeSeq sq = tree_seq(a, b);
  const int L = __builtin_amdgcn_readfirstlane(sq.L), qlen = __builtin_amdgcn_readfirstlane(sq.qlen);
  const int all_steps = __builtin_amdgcn_readfirstlane(sq.steps);
  const int groups = __builtin_amdgcn_readfirstlane(sq.groups);
  if (rg < groups) {  // else no row: the whole workgroup goes on together
  const int whole = all_steps - s_begin;
  const int take = __builtin_amdgcn_readfirstlane(steps_left < whole ? steps_left : whole);
  __syncthreads();  // the LDS of the row group before (or of the prefix) is free
  const bool partial = take < all_steps;
  const int q0 = __builtin_amdgcn_readfirstlane(a.cu_q[b]);
  const int G = a.G;
  const int rows = qlen * G;
  // With one or two units, two waves share each: every step's first 32 keys are the one's, the others the other's.
  const bool split = rows - 32 * kTreeWaves * rg <= 64;  // uniform
  const int part = split ? wave >> 1 : 0;
  const int unit = rg * kTreeWaves + (split ? wave & 1 : wave);
  const bool active = 32 * unit < rows;  // uniform
  // Row 32 unit + i of the sequence: its node and query head (of the last row for those past it).
  struct Row {
    int node, h;
    bool real;
  };
  const FastDiv by_G = a.by_G;
  auto row_of = [&](int i) __attribute__((always_inline)) {
    Row r;
    const int row = 32 * unit + i;
    r.real = row < rows;
    const int x = r.real ? row : rows - 1;
    r.node = x / by_G;
    r.h = kvh * G + x - r.node * G;
    return r;
  };
  const int ctx = __builtin_amdgcn_readfirstlane(sq.ctx);  // the first drafted token's position
  const int seen_by_all = ctx < L ? ctx : L;               // keys before it need no mask
  const int s0 = s_begin, s1 = L > 0 ? s_begin + take : s_begin;

  // Q^T operand j: lane l holds d = 16 j + 8 (l / 32) .. + 7 of row l % 32.
  bf16x8 qb[D / 16];
  {
    const Row r = row_of(n);
    const uint16_t *qp = a.q + static_cast<int64_t>(q0 + r.node) * a.q_st + static_cast<int64_t>(r.h) * a.q_sh;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      u32x4 w = *reinterpret_cast<const u32x4 *>(qp + 16 * j + 8 * hh);
      if (!r.real) w = u32x4{0u, 0u, 0u, 0u};
      qb[j] = __builtin_bit_cast(bf16x8, w);
    }
  }
  const int64_t *const masks = a.mask + static_cast<int64_t>(q0) * a.words;
  const int words = a.words;

  floatx16 o[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[c][r] = 0.f;
  float m_ref = -INFINITY, l_part = 0.f;  // reference maximum (-inf until a key is seen), this lane's share of the sum

  // Copies. Piece p = 64 k + l of a tile's K or V goes to LDS offset 16 p. K: chunk p / 16,
  // token p % 16, as the cache holds it. bf16 V: row p / 2, its token octets in turn (octet 1
  // first in every second eight rows, for the banks); fp8 V: row p.
  const int BS = a.BS, region = D * BS * ESZ, Hkv = a.Hkv, nb = a.nb, Mb = a.Mb;
  const uint8_t *const kc = a.kc, *const vc = a.vc;
  const float *const ksc = a.ksc, *const vsc = a.vsc;
  const float scale_log2 = a.scale_log2;
  const bool stream = a.stream != 0 && groups == 1;  // uniform: nothing reads these keys again
  const uint32_t ldsk0 = lds_addr(ldsk), ldsv0 = lds_addr(ldsv);
  const int32_t *const btrow = a.bt + b * a.bt_stride;
  const FastDiv by_BS = a.by_BS;
  int bix = 64 * s0 / by_BS;  // the block of the next step's first key, and its place there
  int o0 = 64 * s0 - bix * BS;
  const int dbix = 64 / by_BS, do0 = 64 - dbix * BS;
  const int n_blocks = (L + BS - 1) / by_BS;
  // The window: lane i holds the id of block wbase + i. `clean` until a window holds
  // a block that is none (every wave has the same windows).
  int wbase = bix, win;
  bool clean = true;
  auto open_window = [&]() __attribute__((always_inline)) {
    wbase = bix;
    const int l = lane_here();
    win = load_i32_drained(btrow, wbase + l, Mb);
    clean = clean && !__any(wbase + l < n_blocks && !(win >= 0 && win < nb));
  };
  open_window();
  int64_t vbase = 0;  // of the wave's tile of the step whose K went out last: its V
  bool v_ok = false;
  float ks_next = 1.f, vs_next = 1.f, vs_land = 1.f;  // fp8 scales: last K issued, its V, the V that lands next
  bool k_land = false, v_land = false;                // fp8: a tile of this wave's to widen
  // K of the wave's tile of step s into K slot s & 1
  auto issue_k = [&](int s) __attribute__((always_inline)) {
    bool ok = s < s1 && 64 * s + 16 * wave < L;  // uniform
    // (the window holds the next step's blocks too, so that `clean` speaks for it a step ahead;
    // at most once per 56 blocks: its wait drains the copies in flight)
    if (s < s1 && bix - wbase > 56) open_window();
    if (ok) {
      const int ahead = (o0 + 16 * wave) / by_BS, off = o0 + 16 * wave - ahead * BS;
      const int blk = __builtin_amdgcn_readlane(win, bix + ahead - wbase);
      ok = blk >= 0 && blk < nb;
      if (ok) {
        const int64_t rb = static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(blk * Hkv + kvh)) *
                                                static_cast<uint32_t>(region));
        vbase = rb + off * ESZ;
        if constexpr (FP8) {
          ks_next = load_scalar(ksc + blk * Hkv + kvh);
          vs_next = load_scalar(vsc + blk * Hkv + kvh);
        }
        const int l = lane_here();
        const uint32_t lane_k = static_cast<uint32_t>(((l >> 4) * BS + (l & 15)) * 16);
        uint32_t kst = static_cast<uint32_t>(64 * BS);
        asm volatile("" : "+s"(kst));
        const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t *>(wave_uniform(kc + rb + off * 16)), 0, region, kRawBufferWord3);
        const uint32_t dst = __builtin_amdgcn_readfirstlane(ldsk0 + static_cast<uint32_t>((4 * (s & 1) + wave) * TB));
        if (stream)
          buffer_copy16_run_to_lds_nt<NC>(kr, lane_k, kst - 1024u, dst);
        else
          buffer_copy16_run_to_lds<NC>(kr, lane_k, kst - 1024u, dst);
      }
    }
    v_ok = ok;
    k_land = ok;
    if (lane == 0) s_ok[s & 3][wave] = ok ? 1 : 0;
    o0 += do0;
    bix += dbix;
    if (o0 >= BS) {
      o0 -= BS;
      ++bix;
    }
  };
  // V of the wave's tile of step s (whose K went out last) into V slot s & 1
  auto issue_v = [&](int s) __attribute__((always_inline)) {
    v_land = v_ok;
    if (v_ok) {
      vs_land = vs_next;
      const int l = lane_here();
      const uint32_t lane_v = static_cast<uint32_t>(FP8 ? l * BS : (l >> 1) * BS * 2 + 16 * ((l ^ l >> 4) & 1));
      uint32_t vst = static_cast<uint32_t>(64 * BS);
      asm volatile("" : "+s"(vst));
      const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t *>(wave_uniform(vc + vbase)), 0, region, kRawBufferWord3);
      const uint32_t dst = __builtin_amdgcn_readfirstlane(ldsv0 + static_cast<uint32_t>((4 * (s & 1) + wave) * TB));
      if (stream)
        buffer_copy16_run_to_lds_nt<NC>(vr, lane_v, vst - 1024u, dst);
      else
        buffer_copy16_run_to_lds<NC>(vr, lane_v, vst - 1024u, dst);
    }
  };
  // fp8: this wave's landed codes widened in their place. Piece p = 64 i + l of K: chunk
  // p / 16 (16 d) of token p % 16 -> bf16 chunks 2 (p / 16), + 1; of V: row p -> octets
  // 0, 1 of the row. (All of a tile's reads come before its writes: a wave's LDS accesses keep their order.)
  auto widen = [&](int s, auto do_v, auto do_k) __attribute__((always_inline)) {  // V of step s, K of step s + 1
    uint8_t *const tv = ldsv + (4 * (s & 1) + wave) * TB;
    uint8_t *const tk = ldsk + (4 * ((s + 1) & 1) + wave) * TB;
    u32x4 wv[D / 64], wk[D / 64];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      if (do_v) wv[i] = *reinterpret_cast<const u32x4 *>(tv + (64 * i + lane) * 16);
      if (do_k) wk[i] = *reinterpret_cast<const u32x4 *>(tk + (64 * i + lane) * 16);
    }
    asm volatile("" ::: "memory");  // (a lane's writes go over what others read)
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const int p = 64 * i + lane;
      if (do_v) {
        uint8_t *d = tv + p * 32;
        const int first = 2 * (p & 8);  // where the row's octet 0 goes
        *reinterpret_cast<u32x4 *>(d + first) = codes_to_bf16(wv[i][0], wv[i][1], vs_land);
        *reinterpret_cast<u32x4 *>(d + 16 - first) = codes_to_bf16(wv[i][2], wv[i][3], vs_land);
      }
      if (do_k) {
        uint8_t *d = tk + ((2 * (p >> 4)) * 16 + (p & 15)) * 16;
        *reinterpret_cast<u32x4 *>(d) = codes_to_bf16(wk[i][0], wk[i][1], ks_next);
        *reinterpret_cast<u32x4 *>(d + 256) = codes_to_bf16(wk[i][2], wk[i][3], ks_next);
      }
    }
  };
  // V of step s and K of step s + 1 as the products read them. A tile without keys
  // (past the last, or of no block) is masked; its V is zeros, as 0 times what may stand there is not.
  auto land = [&](int s) __attribute__((always_inline)) {
    if (!v_land) {  // uniform
      const int l = lane_here();
      u32x4 *t = reinterpret_cast<u32x4 *>(ldsv + (4 * (s & 1) + wave) * TB);
#pragma unroll
      for (int i = 0; i < TB / 1024; ++i) t[64 * i + l] = u32x4{0u, 0u, 0u, 0u};
    }
    if constexpr (FP8) {
      if (v_land && k_land) {  // uniform: both tiles' reads ahead of the conversions
        widen(s, std::true_type{}, std::true_type{});
      } else {
        if (v_land) widen(s, std::true_type{}, std::false_type{});
        if (k_land) widen(s, std::false_type{}, std::true_type{});
      }
    }
  };

  // Row i of a 32-key half's S^T carries key kperm(i), so that score r of lane
  // l is key 16 (r / 8) + 8 (l / 32) + r % 8 of the half: the PV operand as it stands.
  const int kn = (n & 16) | (((n >> 2) & 3) == 1 ? (n & 3) + 8 : ((n >> 2) & 3) == 2 ? (n & 3) + 4 : (n & 15));
  const bf16x2 ones = __builtin_bit_cast(bf16x2, 0x3F803F80u);
  uint32_t pw[4][4];  // PV operands of the step being finished: packed bf16 probabilities

  // S^T of step s into (x0, x1); of 32 keys (not WHOLE) into x0
  auto qk = [&](int s, floatx16 &x0, floatx16 &x1, auto WHOLE) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 16; ++r) x0[r] = x1[r] = 0.f;
    const uint8_t *lk = ldsk + ((s & 1) * 4 + 2 * (WHOLE ? 0 : part) + (kn >> 4)) * TB + (kn & 15) * 16;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      const bf16x8 a0 = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(lk + (2 * j + hh) * 256));
      x0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a0, qb[j], x0, 0, 0, 0);
      if constexpr (WHOLE) {
        const bf16x8 a1 = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4 *>(lk + 2 * TB + (2 * j + hh) * 256));
        x1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a1, qb[j], x1, 0, 0, 0);
      }
    }
  };
  // The tiles of step s that hold keys, a bit each.
  auto tiles = [&](int s) __attribute__((always_inline)) {
    const u32x4 w = *reinterpret_cast<const u32x4 *>(s_ok[s & 3]);
    return __builtin_amdgcn_readfirstlane(w[0] | w[1] << 1 | w[2] << 2 | w[3] << 3);
  };
  // The keys of step s that this lane's row sees, a bit each.
  auto window = [&](int s, uint32_t ok) __attribute__((always_inline)) {
    const int kb = 64 * s, first = kb - ctx;  // the node of the step's first key
    uint64_t seen = ~0ull;
    if (first > -64) {
      const Row r = row_of(lane_here() & 31);
      auto word = [&](int i) __attribute__((always_inline)) {
        return r.real && i < words ? static_cast<uint64_t>(masks[r.node * words + i]) : 0ull;
      };
      if (first < 0) {
        seen = ((1ull << -first) - 1ull) | (word(0) << -first);
      } else {
        const int w = first >> 6, sh = first & 63;
        seen = word(w) >> sh;
        if (sh) seen |= word(w + 1) << (64 - sh);
      }
    }
    const int left = L - kb;
    if (left < 64) seen &= (1ull << left) - 1ull;
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (!(ok >> t & 1)) seen &= ~(0xFFFFull << (16 * t));
    return seen;
  };
  // Exponents against the reference maximum (0 before the first seen key).
  auto expo = [&](floatx16 &x0, floatx16 &x1, auto WHOLE) __attribute__((always_inline)) {
    const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x0[r] = __builtin_fmaf(x0[r], scale_log2, -m_use);
      if constexpr (WHOLE) x1[r] = __builtin_fmaf(x1[r], scale_log2, -m_use);
    }
  };
  auto hide = [&](uint64_t seen, floatx16 &x0, floatx16 &x1, auto WHOLE) __attribute__((always_inline)) {
    const uint64_t v = seen >> (8 * (lane_here() >> 5) + (WHOLE ? 0 : 32 * part));
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if (!(v >> (16 * (r >> 3) + (r & 7)) & 1)) x0[r] = -INFINITY;
      if constexpr (WHOLE)
        if (!(v >> (32 + 16 * (r >> 3) + (r & 7)) & 1)) x1[r] = -INFINITY;
    }
  };
  auto largest = [&](const floatx16 &x0, const floatx16 &x1, auto WHOLE) __attribute__((always_inline)) {
    float mt = fmaxf(x0[0], x0[1]), mt1 = fmaxf(x1[0], x1[1]);
#pragma unroll
    for (int r = 2; r < 16; r += 2) {
      mt = fmaxf(fmaxf(mt, x0[r]), x0[r + 1]);
      if constexpr (WHOLE) mt1 = fmaxf(fmaxf(mt1, x1[r]), x1[r + 1]);
    }
    if constexpr (WHOLE) mt = fmaxf(mt, mt1);
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
    return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
  };
  // The rare move of the reference maximum (after the PV products of the steps before).
  auto rescale = [&](float mt, floatx16 &x0, floatx16 &x1, auto WHOLE) __attribute__((always_inline)) {
    const bool unset = m_ref == -INFINITY;
    const bool move = unset ? mt > -INFINITY : mt > SOFTMAX_TAU;
    if (__any(move)) {
      asm volatile("");  // stays a branch: a step seldom has it
      const float sh = move ? mt : 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        x0[r] -= sh;
        if constexpr (WHOLE) x1[r] -= sh;
      }
      const float corr = move && !unset ? fast_exp2(-sh) : 1.f;
      l_part *= corr;
      if (move) m_ref = unset ? sh : m_ref + sh;
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[c][r] *= corr;
    }
  };
  // Probabilities, packed as the PV operands, and the sum of the rounded ones.
  auto probs = [&](floatx16 &x0, floatx16 &x1, auto WHOLE) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      x0[r] = fast_exp2(x0[r]);
      if constexpr (WHOLE) x1[r] = fast_exp2(x1[r]);
    }
    float ps = 0.f;
#pragma unroll
    for (int t = 0; t < (WHOLE ? 4 : 2); ++t) {
      const floatx16 &sv = t < 2 ? x0 : x1;
      const int e0 = 8 * (t & 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pw[t][i] = pack_bf16x2(sv[e0 + 2 * i], sv[e0 + 2 * i + 1]);
        ps = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pw[t][i]), ones, ps, false);
      }
    }
    l_part += ps;
  };
  // P V^T of step s
  auto pv = [&](int s, auto WHOLE) __attribute__((always_inline)) {
    const uint8_t *lv = ldsv + ((s & 1) * 4 + 2 * (WHOLE ? 0 : part)) * TB + n * 32 + 16 * (hh ^ ((n >> 3) & 1));
#pragma unroll
    for (int t = 0; t < (WHOLE ? 4 : 2); ++t) {
      const bf16x8 pb = __builtin_bit_cast(bf16x8, (u32x4{pw[t][0], pw[t][1], pw[t][2], pw[t][3]}));
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(lv + t * TB + 1024 * c);
        o[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, w), pb, o[c], 0, 0, 0);
      }
    }
  };
  // The same of a step that masks: slots past the last token (they may hold
  // anything) as zeros. V that are not finite are zeros there too, and are added
  // to the rows that see their keys: as many +inf, -inf or both (a NaN) as products of
  // where they stand with what is seen count.
  auto pv_masked = [&](int s, auto WHOLE) __attribute__((always_inline)) {
    const int l = lane_here(), n = l & 31, hh = l >> 5;
    const int t0 = WHOLE ? 0 : 2 * part;
    const uint8_t *const lv = ldsv + ((s & 1) * 4 + t0) * TB + n * 32 + 16 * (hh ^ ((n >> 3) & 1));
    bool odd = false;
#pragma unroll
    for (int t = 0; t < (WHOLE ? 4 : 2); ++t) {
      const int left = L - 64 * s - 16 * (t0 + t);
      if (left <= 0) continue;  // uniform
      u32x4 w[D / 32];
#pragma unroll
      for (int c = 0; c < D / 32; ++c) w[c] = *reinterpret_cast<const u32x4 *>(lv + t * TB + 1024 * c);
      if (left < 16) {  // uniform
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[c][i] &= (8 * hh + 2 * i < left ? 0xFFFFu : 0u) | (8 * hh + 2 * i + 1 < left ? 0xFFFF0000u : 0u);
      }
      u16x2 most = {0, 0};  // largest magnitude bits
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, w[c][i] & 0x7FFF7FFFu));
      if (__any(most[0] >= 0x7F80u || most[1] >= 0x7F80u)) {
        odd = true;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[c][i] &= ((w[c][i] & 0x7F80u) == 0x7F80u ? 0u : 0xFFFFu) |
                       ((w[c][i] & 0x7F800000u) == 0x7F800000u ? 0u : 0xFFFF0000u);
      }
      const bf16x8 pb = __builtin_bit_cast(bf16x8, (u32x4{pw[t][0], pw[t][1], pw[t][2], pw[t][3]}));
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
        o[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, w[c]), pb, o[c], 0, 0, 0);
    }
    if (!odd) return;  // uniform
    const uint64_t seen = window(s, tiles(s)) >> (8 * hh + 16 * t0);
#pragma unroll 1
    for (int t = 0; t < (WHOLE ? 4 : 2); ++t) {
      u32x4 vis;  // 1 where the row sees the key
#pragma unroll
      for (int i = 0; i < 4; ++i)
        vis[i] = (seen >> (16 * t + 2 * i) & 1 ? 0x3F80u : 0u) | (seen >> (16 * t + 2 * i + 1) & 1 ? 0x3F800000u : 0u);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(lv + t * TB + 1024 * c);
#pragma unroll
        for (int sign = 0; sign < 2; ++sign) {  // 1 where V is a NaN or the infinity of this sign
          const uint32_t inf = sign ? 0xFF80u : 0x7F80u;
          u32x4 is;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t lo = w[i] & 0xFFFFu, hi = w[i] >> 16;
            is[i] = ((lo & 0x7FFFu) > 0x7F80u || lo == inf ? 0x3F80u : 0u) |
                    ((hi & 0x7FFFu) > 0x7F80u || hi == inf ? 0x3F800000u : 0u);
          }
          floatx16 x;
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = 0.f;
          x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, is), __builtin_bit_cast(bf16x8, vis), x,
                                                      0, 0, 0);
#pragma unroll
          for (int r = 0; r < 16; ++r) o[c][r] += x[r] > 0.f ? (sign ? -INFINITY : INFINITY) : 0.f;
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  };

  // The copies' turn of step s, and the next ones on their way.
  auto turn = [&](int s) __attribute__((always_inline)) {
    wait_vmcnt<0>();  // this wave's copies of step s's V and step s + 1's K
    land(s);
    barrier_lds();    // ... every wave's; every wave is done with step s - 1
    issue_v(s + 1);
    issue_k(s + 2);
  };
  // Step s finished while step s + 1 is scored, both of whole tiles of the context.
  auto body = [&](int s, floatx16 &c0, floatx16 &c1, floatx16 &n0, floatx16 &n1, auto WHOLE)
                  __attribute__((always_inline)) {
    turn(s);
    if (!active) return;  // uniform
    qk(s + 1, n0, n1, WHOLE);
    probs(c0, c1, WHOLE);
    // keeps the probabilities in this block
    if constexpr (WHOLE)
      asm volatile("" ::"v"(l_part), "v"(pw[0][0]), "v"(pw[0][1]), "v"(pw[0][2]), "v"(pw[0][3]), "v"(pw[1][0]),
                   "v"(pw[1][1]), "v"(pw[1][2]), "v"(pw[1][3]), "v"(pw[2][0]), "v"(pw[2][1]), "v"(pw[2][2]),
                   "v"(pw[2][3]), "v"(pw[3][0]), "v"(pw[3][1]), "v"(pw[3][2]), "v"(pw[3][3]));
    else
      asm volatile("" ::"v"(l_part), "v"(pw[0][0]), "v"(pw[0][1]), "v"(pw[0][2]), "v"(pw[0][3]), "v"(pw[1][0]),
                   "v"(pw[1][1]), "v"(pw[1][2]), "v"(pw[1][3]));
    // the score products of step s + 1 interleaved with step s's probabilities
    constexpr int QK = (WHOLE ? 2 : 1) * D / 16, PV = (WHOLE ? 4 : 2) * D / 32;  // products
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);  // LDS reads, four ahead
#pragma unroll
    for (int i = 0; i < QK; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
      if (i + 4 < QK) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS read
      __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);  // VALU
    }
    expo(n0, n1, WHOLE);
    const float mt = largest(n0, n1, WHOLE);
    pv(s, WHOLE);
    // step s's PV products interleaved with step s + 1's exponents
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < PV; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (i + 4 < PV) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
    }
    rescale(mt, n0, n1, WHOLE);
  };

  auto keys = [&](auto WHOLE) __attribute__((always_inline)) {
    issue_k(s0);
    if constexpr (FP8) {
      wait_vmcnt<0>();
      if (k_land) widen(s0 - 1, std::false_type{}, std::true_type{});
    }
    issue_v(s0);
    issue_k(s0 + 1);
    if constexpr (!FP8) {  // K of step s0 landed: at most its V and the next K on their way
      if (k_land) wait_vmcnt<2 * NC>(); else wait_vmcnt<NC>();
      if (!v_land) wait_vmcnt<0>();  // (no tile of step s0)
    }
    barrier_lds();
    constexpr int QK = (WHOLE ? 2 : 1) * D / 16;
    floatx16 a0, a1;
    auto score = [&](int s) __attribute__((always_inline)) {
      qk(s, a0, a1, WHOLE);
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);  // LDS reads four ahead of their MFMAs, not all at once
#pragma unroll
      for (int i = 0; i < QK; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (i + 4 < QK) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      expo(a0, a1, WHOLE);
      const uint32_t ok = tiles(s);
      if (ok != 15u || 64 * s + 64 > seen_by_all) {  // uniform
        hide(window(s, ok), a0, a1, WHOLE);
      }
      rescale(largest(a0, a1, WHOLE), a0, a1, WHOLE);
    };
    if (active) score(s0);
    // Steps of context alone, in pairs: what a pair scores, steps s + 1 and s + 2, is of
    // windows opened before it.
    int s = s0;
    {
      floatx16 b0, b1;
      const int ends = (seen_by_all >> 6) < s1 ? (seen_by_all >> 6) : s1;
      for (; s + 2 < ends && clean; s += 2) {
        body(s, a0, a1, b0, b1, WHOLE);
        body(s + 1, b0, b1, a0, a1, WHOLE);
      }
      if (s + 1 < ends && clean) {
        body(s, a0, a1, b0, b1, WHOLE);
        ++s;
        a0 = b0;
        a1 = b1;
      }
    }
    // The others, one at a time.
#pragma unroll 1
    for (; s < s1; ++s) {
      turn(s);
      if (!active) continue;  // uniform
      probs(a0, a1, WHOLE);
      pv_masked(s, WHOLE);
      if (s + 1 < s1) score(s + 1);
    }
  };
  if (s1 > s0) {
    if (split) keys(std::false_type{}); else keys(std::true_type{});
  }
  bool writes = active;
  if (split) {  // the second part's waves hand theirs to the first's
    barrier_lds();
    float *const jo = reinterpret_cast<float *>(unit & 1 ? ldsv : ldsk);
    const int l = lane_here();
    if (active && part == 1) {
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<floatx4 *>(jo + ((4 * c + g) * 64 + l) * 4) =
              floatx4{o[c][4 * g], o[c][4 * g + 1], o[c][4 * g + 2], o[c][4 * g + 3]};
      jo[32 * D + l] = m_ref;
      jo[32 * D + 64 + l] = l_part;
    }
    barrier_lds();
    writes = active && part == 0;
    if (writes) {
      const float mb = jo[32 * D + l], m = fmaxf(m_ref, mb), m_use = m == -INFINITY ? 0.f : m;
      const float wa = fast_exp2(m_ref - m_use), wb = fast_exp2(mb - m_use);  // 0 of a part that saw no key
      l_part = l_part * wa + jo[32 * D + 64 + l] * wb;
      m_ref = m;
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const floatx4 x = *reinterpret_cast<const floatx4 *>(jo + ((4 * c + g) * 64 + l) * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[c][4 * g + e] = o[c][4 * g + e] * wa + x[e] * wb;
        }
    }
  }
  const TreeArgs &ae = tree_args();
  if (writes) {
  const int lane = lane_here(), n = lane & 31, hh = lane >> 5;
  float l = l_part;
  {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  if (partial) {  // uniform
    const int64_t slot = 2 * s_place + (later ? 1 : 0);
    float *pp = ae.part + (slot * kTreeWaves + wave) * tree_part_floats<D>();
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
  } else if (const Row r = row_of(n); r.real) {
    const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
    if (ae.sinks != nullptr) l += exp2f(ae.sinks[r.h] * 1.4426950408889634f - m_use);
    const float inv = l != 0.f ? 1.f / l : 0.f;
    uint16_t *const op = ae.out + static_cast<int64_t>(q0 + r.node) * ae.o_st + static_cast<int64_t>(r.h) * ae.o_sh;
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g)  // d = 32 c + 8 g + 4 hh + 0..3
        *reinterpret_cast<u32x2 *>(op + 32 * c + 8 * g + 4 * hh) =
            u32x2{pack_bf16x2(o[c][4 * g] * inv, o[c][4 * g + 1] * inv),
                  pack_bf16x2(o[c][4 * g + 2] * inv, o[c][4 * g + 3] * inv)};
  }
  }
  if (partial && s_begin == 0 && threadIdx.x == 0) {  // the group's first part (and the last of this share)
    const TreeShare share = s_share;
    const int w = s_place;
    const int w1 = share.of(share.begin(w + 1) + (all_steps - take) - 1);  // the workgroup of the group's last step
    tree_counts<D>(ae.part)[id] = w1 - w + 1;
    tree_records<D>(ae.part)[id] = TreeRec{2 * w + (later ? 1 : 0), 2 * (w + 1), b, kvh, rg, {0, 0, 0}};
  }
  steps_left -= take;
  later = true;
  }
  if (steps_left <= 0) break;
  s_begin = 0;
  const TreeArgs &an = tree_args();
  if (++rg >= groups) {
    rg = 0;
    if (++b == an.batch) {
      b = 0;
      if (++kvh == an.Hkv) break;  // never with steps left
    }
  }
  }
}

// Log-sum-exp merge of the cut row groups' parts. A wave takes 8 output columns
// of a unit at a time, of the records that name a group in turn over the grid's waves:
// each wave finds them by itself in the list of the part counts. (A workgroup per
// record instead, three quarters of which are empty, cost 8 us for their dispatch alone.)
// 256 / 512 / 1,024 / 2,048 workgroups: 64 sequences of 100 to 8,000 tokens with 16 to 48 drafted
// 333 / 313 / 304 / 303 us with their attention; a merge of nothing costs the same.
constexpr int kMergeGroups = 1024;
template <int D>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
  constexpr int PF = tree_part_floats<D>();
  constexpr int CG = D / 8;  // column groups
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int lane = threadIdx.x & 63, n = lane & 31, hh = lane >> 5;
  const int *counts = tree_counts<D>(a.part);
  uint64_t named[kTreeShare / 64];
  int total = 0;
#pragma unroll
  for (int i = 0; i < kTreeShare / 64; ++i) named[i] = __ballot(counts[64 * i + lane] > 0);
#pragma unroll
  for (int i = 0; i < kTreeShare / 64; ++i) total += __builtin_popcountll(named[i]);
  total *= kTreeWaves * CG;
  for (int item = blockIdx.x * 4 + wave; item < total; item += kMergeGroups * 4) {
    int k = item / (kTreeWaves * CG), id = 0;  // the k-th record that names a group
    uint64_t bits = 0;
#pragma unroll
    for (int i = 0; i < kTreeShare / 64; ++i) {
      const int c = __builtin_popcountll(named[i]);
      if (k >= 0 && k < c) {
        id = 64 * i;
        bits = named[i];
        for (; k > 0; --k) bits &= bits - 1;
        k = 0;
      }
      k -= c;
    }
    id = __builtin_amdgcn_readfirstlane(id + __builtin_ctzll(bits));
    const int unit = item / CG % kTreeWaves, cg = item % CG;
    const int parts = __builtin_amdgcn_readfirstlane(counts[id]);
    const TreeRec rec = tree_records<D>(a.part)[id];
    const int q0 = a.cu_q[rec.b], rows = (a.cu_q[rec.b + 1] - q0) * a.G;
    const int row = 32 * (rec.group * kTreeWaves + unit) + n;
    const float *p0 = a.part + (static_cast<int64_t>(rec.slot) * kTreeWaves + unit) * PF;
    const float *pn = a.part + (static_cast<int64_t>(rec.next) * kTreeWaves + unit) * PF;
    constexpr int64_t step = 2 * kTreeWaves * PF;
    if (row - n >= rows) continue;
    float M = -INFINITY, l = 0.f;
    floatx4 acc = {0.f, 0.f, 0.f, 0.f};
    constexpr int N = 8;  // parts in flight: a long group has tens
    for (int i0 = 0; i0 < parts; i0 += N) {
      float m[N], s[N];
      floatx4 x[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        m[j] = -INFINITY;
        if (i0 + j < parts) {  // uniform
          const float *ps = i0 + j == 0 ? p0 : pn + (i0 + j - 1) * step;
          m[j] = ps[32 * D + n];
          s[j] = ps[32 * D + 32 + n];
          x[j] = *reinterpret_cast<const floatx4 *>(ps + (cg * 64 + lane) * 4);
        }
      }
      float top = M;
#pragma unroll
      for (int j = 0; j < N; ++j) top = fmaxf(top, m[j]);
      const float m_use = top == -INFINITY ? 0.f : top;
      const float was = exp2f(M - m_use);  // 0 while no part saw a key
      l *= was;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] *= was;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (i0 + j < parts) {
          const float w = exp2f(m[j] - m_use);  // 0 for a part of which the row saw no key
          l += w * s[j];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] += w * x[j][e];
        }
      }
      M = top;
    }
    if (row >= rows) continue;
    const int node = row / a.by_G, h = rec.kvh * a.G + row - node * a.G;
    const float m_use = M == -INFINITY ? 0.f : M;
    if (a.sinks != nullptr) l += exp2f(a.sinks[h] * 1.4426950408889634f - m_use);
    const float inv = l != 0.f ? 1.f / l : 0.f;
    uint16_t *op = a.out + static_cast<int64_t>(q0 + node) * a.o_st + static_cast<int64_t>(h) * a.o_sh;
    *reinterpret_cast<u32x2 *>(op + 8 * cg + 4 * hh) =
        u32x2{pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv)};
  }
}

// The workgroups that share a launch; 0: one per row group. Contexts of at most twelve steps are
// not cut, and a line of 2^31 steps is not formed. Whole / cut, with the merge's launch, us, at 500, 800 and
// 1,200 tokens, 32 and 8 heads of 128: one sequence with 8 drafted 20 / 25, 23 / 25, 29 / 25 (fp8
// 18 / 18, 24 / 22, 32 / 23), with 128 29 / 30, 36 / 32, 45 / 35; eight with 16 22 / 30, 26 / 31, 33 / 35; 14
// and 2 heads of 64, one with 8: 21 / 25, 20 / 25, 23 / 25.
static int tree_sharing(int batch, int Hkv, int G, int max_query_len, int max_seq) {
  const int64_t steps = (static_cast<int64_t>(max_seq) + 63) / 64;
  const int64_t groups = (static_cast<int64_t>(max_query_len) * G + kTreeRows - 1) / kTreeRows;
  return steps > 12 && groups * batch <= INT32_MAX / (steps * Hkv) ? kTreeShare : 0;
}

static int64_t tree_workspace(int share, int D) {
  return share > 0 ? static_cast<int64_t>(share) * (2 * kTreeWaves * (32 * D + 64) * 4 + 4 + sizeof(TreeRec)) : 0;
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
  return tree_workspace(
      tree_sharing(batch, num_kv_heads, num_q_heads / num_kv_heads, max_query_len, max_seq_len), head_dim);
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
  WKV_CHECK_ARG(max_query_len > 0 && max_seq_len >= 0 && max_seq_len <= INT32_MAX - 256,
                "max_query_len must be > 0 and max_seq_len in [0, 2^31 - 257]");
  WKV_CHECK_ARG(tree_mask != nullptr && reinterpret_cast<uintptr_t>(tree_mask) % 8 == 0, "tree_mask must be non-NULL int64");
  WKV_CHECK_ARG(mask_words >= 1 && mask_words <= WKV_TREE_MAX_WORDS, "mask_words must be in [1, %d] (got %d)",
                WKV_TREE_MAX_WORDS, mask_words);
  WKV_CHECK_ARG(std::isfinite(scale), "scale must be finite");
  WKV_CHECK_ARG(reinterpret_cast<uintptr_t>(sinks) % 4 == 0, "sinks must be fp32");
  WKV_CHECK_ARG(static_cast<int64_t>(max_query_len) * G <= (1 << 24), "max_query_len * query heads per KV head too large");
  const int64_t table_tokens = static_cast<int64_t>(max_blocks_per_seq) * BS;
  const int max_seq = max_seq_len < table_tokens ? max_seq_len : static_cast<int>(table_tokens);
  const int share = workspace != nullptr ? tree_sharing(batch, Hkv, G, max_query_len, max_seq) : 0;
  const int64_t need = tree_workspace(share, D);
  if (need > 0)
    WKV_CHECK_ARG(aligned16(workspace) && workspace_bytes >= need, "workspace too small: need %lld bytes, got %lld",
                  (long long)need, (long long)workspace_bytes);
  const int64_t items = static_cast<int64_t>(batch) * Hkv;
  const int groups = static_cast<int>((static_cast<int64_t>(max_query_len) * G + kTreeRows - 1) / kTreeRows);
  // (A shared launch may turn out to be of whole row groups: as many workgroups as there can be, to a limit.)
  const int64_t most = (items * groups + 7) / 8 * 8;
  const int64_t n_wg = share == 0     ? (items + 7) / 8 * 8 * groups
                       : most < share ? share
                                      : (most < kTreeMost ? most : kTreeMost);
  WKV_CHECK_ARG(n_wg <= INT32_MAX / kTreeThreads, "too many sequences, KV heads and drafted tokens");
  rc = append();
  if (rc) return rc;
  TreeArgs a{};
  a.kc = static_cast<const uint8_t *>(cache->k);
  a.vc = static_cast<const uint8_t *>(cache->v);
  a.ksc = cache->k_scale;
  a.vsc = cache->v_scale;
  a.q = static_cast<const uint16_t *>(q);
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.out = static_cast<uint16_t *>(out);
  a.o_st = out_stride_t;
  a.o_sh = out_stride_h;
  a.cu_q = cu_seqlens_q;
  a.seq_lens = seq_lens;
  a.bt = block_table;
  a.bt_stride = bt_stride;
  a.mask = tree_mask;
  a.words = mask_words;
  a.batch = batch;
  a.Mb = max_blocks_per_seq;
  a.max_seq = max_seq;
  a.Hkv = Hkv;
  a.G = G;
  a.BS = BS;
  a.nb = static_cast<int>(cache->num_blocks);
  a.by_BS = fast_div(BS);
  a.by_G = fast_div(G);
  a.share = share;
  a.groups = groups;
  a.stream = (cache->flags & WKV_CACHE_SHARED_BLOCKS) == 0;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.part = static_cast<float *>(workspace);
  a.sinks = sinks;
  const dim3 grid(static_cast<unsigned>(n_wg));
  auto s = static_cast<hipStream_t>(stream);
  const bool fp8 = cache->kv_dtype == WKV_KV_FP8_E4M3;
#define WKV_TREE(Dv, F8) tree_gqa_kernel<Dv, F8><<<grid, kTreeThreads, 0, s>>>(a)
  if (D == 128) {
    if (fp8) WKV_TREE(128, true); else WKV_TREE(128, false);
  } else {
    if (fp8) WKV_TREE(64, true); else WKV_TREE(64, false);
  }
#undef WKV_TREE
  WKV_CHECK_LAUNCH("tree attention");
  if (share > 0) {
    if (D == 128)
      tree_merge_kernel<128><<<kMergeGroups, 256, 0, s>>>(a);
    else
      tree_merge_kernel<64><<<kMergeGroups, 256, 0, s>>>(a);
    WKV_CHECK_LAUNCH("tree attention merge");
  }
  return WKV_OK;
}
