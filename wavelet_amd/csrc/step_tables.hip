// A step's bookkeeping on the GPU (gfx950): block tables, slots, positions and
// tree masks from the request lengths (wkv_extend_tables), and the accepted
// path of a verified tree (wkv_accept_tree). Both are bound by their launch and
// a few dependent round trips, not by bytes: 16 bytes per token and 24 per
// sequence. 64 sequences with trees of 16 nodes 7.9 us, with 75,000 prompt tokens
// 8.4 + 4.2 us (two launches); the paths of 256 trees of 64 nodes 4.0 us.
#include "wkv_common.h"

namespace wkv {

constexpr int kTablesThreads = 1024;
constexpr int kTablesPer = WKV_STEP_MAX_BATCH / kTablesThreads;  // sequences per thread
// Rows that the planning workgroup writes itself (four per thread); more go to
// a second launch over the chip.
constexpr int kTablesOwnRows = 4096;

struct TablesArgs {
  int32_t *table;
  int64_t table_stride;
  int width;
  const int32_t *held, *seq_lens, *new_lens, *free_blocks, *taken;
  int32_t num_free;
  int B, BS, rows;
  const int32_t *parents;
  int words;
  int limit;  // cached and new tokens of a sequence
  int32_t *held_out, *taken_out, *context, *cu, *refused;
  int64_t *slots, *positions, *masks;
};

// Inclusive sum over the workgroup, held at `cap` (non-negative terms, all <= cap:
// a held sum stays held, so the order of the additions does not matter).
__device__ __forceinline__ uint32_t held_scan(uint32_t x, uint32_t cap, uint32_t *red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o, 64);
    if (lane >= o) x = min(x + y, cap);
  }
  __syncthreads();  // the sums of the scan before
  if (lane == 63) red[wave] = x;
  __syncthreads();
  uint32_t base = 0;
#pragma unroll
  for (int w = 0; w < kTablesThreads / 64; ++w)
    if (w < wave) base = min(base + red[w], cap);
  return min(base + x, cap);
}

// The last entry i of s[0 .. n] (rising) with s[i] <= x; s[0] <= x < s[n].
template <class P>
__device__ __forceinline__ int last_at_most(const P s, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// One row's outputs: token j of a sequence with L cached tokens whose first row
// is `first`, in block `block`. Trees: the walk to the root
// gives the depth and the mask. A parent is an earlier node, so the walk ends.
__device__ __forceinline__ void write_row(const TablesArgs &a, int r, int first, int j, int L, int block, bool real) {
  int64_t slot = -1, at = -1;
  uint64_t m[WKV_TREE_MAX_WORDS] = {};
  if (real) {
    at = L + j;
    if (block >= 0) slot = static_cast<int64_t>(block) * a.BS + (L + j) % a.BS;
    if (a.words > 0) {
      int depth = 0;
      for (int i = j;;) {
#pragma unroll
        for (int w = 0; w < WKV_TREE_MAX_WORDS; ++w)
          if (i >> 6 == w) m[w] |= 1ull << (i & 63);
        const int p = a.parents[first + i];
        if (p < 0 || p >= i) break;
        i = p;
        ++depth;
      }
      at = L + depth;
    }
  }
  a.slots[r] = slot;
  a.positions[r] = at;
#pragma unroll
  for (int w = 0; w < WKV_TREE_MAX_WORDS; ++w)
    if (w < a.words) a.masks[static_cast<int64_t>(r) * a.words + w] = static_cast<int64_t>(m[w]);
}

// One workgroup: the sums over the sequences (rows, blocks), who is granted its
// blocks, the new table entries and, with ROWS, every row. What it reads of
// held and taken is read before the first write (they may be the outputs).
template <bool ROWS>
__global__ __launch_bounds__(kTablesThreads) void tables_plan_kernel(TablesArgs a) {
  __shared__ uint32_t red[kTablesThreads / 64];
  __shared__ int s_cu[WKV_STEP_MAX_BATCH + 1], s_need[WKV_STEP_MAX_BATCH + 1];  // sums before each sequence
  __shared__ int s_held[WKV_STEP_MAX_BATCH], s_len[WKV_STEP_MAX_BATCH];         // length, -1: nothing granted
  __shared__ int s_refused, s_given;
  const int b0 = threadIdx.x * kTablesPer;
  const int taken = max(*a.taken, 0);
  if (threadIdx.x == 0) s_refused = s_given = 0;
  int L[kTablesPer], n[kTablesPer], held[kTablesPer];
  const uint32_t row_cap = static_cast<uint32_t>(a.rows) + 1u;
  uint32_t sum = 0;
#pragma unroll
  for (int k = 0; k < kTablesPer; ++k) {
    const int b = b0 + k;
    const bool in = b < a.B;
    L[k] = in ? max(a.seq_lens[b], 0) : 0;
    n[k] = in ? max(a.new_lens[b], 0) : 0;
    held[k] = in ? max(a.held[b], 0) : 0;
    sum = min(sum + min(static_cast<uint32_t>(n[k]), row_cap), row_cap);
  }
  uint32_t before = held_scan(sum, row_cap, red);
  // (the exclusive sum again from the sequences before: a held sum cannot be taken apart)
  const uint32_t prev_rows = __shfl_up(before, 1, 64);
  __shared__ uint32_t tail[kTablesThreads / 64];
  if ((threadIdx.x & 63) == 63) tail[threadIdx.x >> 6] = before;
  __syncthreads();
  uint32_t row = (threadIdx.x & 63) ? prev_rows : (threadIdx.x ? tail[(threadIdx.x >> 6) - 1] : 0u);
  uint32_t need[kTablesPer];
  bool fits[kTablesPer];
  const uint32_t need_cap = static_cast<uint32_t>(a.num_free) + 1u;
  sum = 0;
#pragma unroll
  for (int k = 0; k < kTablesPer; ++k) {
    const int b = b0 + k;
    if (b < a.B) s_cu[b] = static_cast<int>(min(row, static_cast<uint32_t>(a.rows)));
    row = min(row + min(static_cast<uint32_t>(n[k]), row_cap), row_cap);
    if (b == a.B - 1) s_cu[a.B] = static_cast<int>(min(row, static_cast<uint32_t>(a.rows)));
    const int64_t end = static_cast<int64_t>(L[k]) + n[k], total = (end + a.BS - 1) / a.BS;
    fits[k] = n[k] > 0 && total <= a.width && end <= a.limit && row <= static_cast<uint32_t>(a.rows) &&
              (a.words == 0 || n[k] <= 64 * a.words);
    need[k] = fits[k] && total > held[k] ? min(static_cast<uint32_t>(total - held[k]), need_cap) : 0u;
    sum = min(sum + need[k], need_cap);
  }
  before = held_scan(sum, need_cap, red);
  const uint32_t prev_need = __shfl_up(before, 1, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) tail[threadIdx.x >> 6] = before;
  __syncthreads();
  uint32_t asked = (threadIdx.x & 63) ? prev_need : (threadIdx.x ? tail[(threadIdx.x >> 6) - 1] : 0u);
  int given = 0, refused = 0;
#pragma unroll
  for (int k = 0; k < kTablesPer; ++k) {
    const int b = b0 + k;
    if (b < a.B) {
      // (the blocks asked for so far and those taken before fit the list)
      const uint32_t start = asked;
      asked = min(asked + need[k], need_cap);
      const bool granted =
          fits[k] && (need[k] == 0 || static_cast<int64_t>(taken) + asked <= static_cast<int64_t>(a.num_free));
      s_need[b] = static_cast<int>(start);
      s_held[b] = held[k];
      s_len[b] = granted ? L[k] : -1;
      if (granted) given += static_cast<int>(need[k]);
      if (n[k] > 0 && !granted) ++refused;
      a.context[b] = n[k] == 0 ? L[k] : (granted ? L[k] + n[k] : 0);
      a.held_out[b] = held[k] + (granted ? static_cast<int>(need[k]) : 0);
      a.cu[b] = s_cu[b];
      if (b == a.B - 1) {
        s_need[a.B] = static_cast<int>(asked);
        a.cu[a.B] = s_cu[a.B];
      }
    }
  }
  if (given) atomicAdd(&s_given, given);
  if (refused) atomicAdd(&s_refused, refused);
  __syncthreads();
  if (threadIdx.x == 0) {
    *a.taken_out = taken + s_given;
    *a.refused = s_refused;
  }
  // New table entries: free block `taken + x` of the asked ones, in batch order.
  const int asked_all = s_need[a.B];
  for (int x = threadIdx.x; x < asked_all; x += kTablesThreads) {
    if (static_cast<int64_t>(taken) + x >= a.num_free) break;
    const int b = last_at_most(s_need, a.B, x);
    if (s_len[b] >= 0)
      a.table[b * a.table_stride + s_held[b] + (x - s_need[b])] = a.free_blocks[taken + x];
  }
  if constexpr (ROWS) {
    for (int r = threadIdx.x; r < a.rows; r += kTablesThreads) {
      const bool in = r < s_cu[a.B];
      const int b = in ? last_at_most(s_cu, a.B, r) : 0;
      const int j = r - s_cu[b], len = s_len[b];
      const bool real = in && len >= 0;
      int block = -1;
      if (real) {  // (an entry that this call makes comes from the list, not from the table)
        const int i = (len + j) / a.BS;
        block = i < s_held[b] ? a.table[b * a.table_stride + i] : a.free_blocks[taken + s_need[b] + (i - s_held[b])];
      }
      write_row(a, r, s_cu[b], j, len, block, real);
    }
  }
}

// The rows of a larger step, after the plan: one thread each.
__global__ __launch_bounds__(256) void tables_rows_kernel(TablesArgs a) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= a.rows) return;
  const bool in = r < a.cu[a.B];
  const int b = in ? last_at_most(a.cu, a.B, r) : 0;
  const int first = a.cu[b], j = r - first;
  const bool real = in && a.context[b] > 0;  // a sequence with rows that was granted them
  const int L = max(a.seq_lens[b], 0);
  const int block = real ? a.table[b * a.table_stride + (L + j) / a.BS] : -1;
  write_row(a, r, first, j, L, block, real);
}

// One wave per sequence: its nodes four to a lane, the path entry of depth i in
// lane i. Each step compares every node at once with the current one.
__global__ __launch_bounds__(256) void accept_tree_kernel(const int64_t *__restrict__ draft,
                                                          const int32_t *__restrict__ parents,
                                                          const int64_t *__restrict__ target, int rows,
                                                          const int32_t *__restrict__ cu, const int32_t *seq_lens,
                                                          const int32_t *__restrict__ context, int B, int max_depth,
                                                          int32_t *__restrict__ accepted, int32_t *__restrict__ path,
                                                          int64_t *__restrict__ next, int32_t *len_out,
                                                          int64_t *__restrict__ pending) {
  constexpr int N = WKV_TREE_MAX_WORDS;
  const int b = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x * 4 + (threadIdx.x >> 6)));
  if (b >= B) return;
  const int lane = threadIdx.x & 63;
  const int q0 = min(max(cu[b], 0), rows), L = max(seq_lens[b], 0);
  int n = min(cu[b + 1], rows) - q0;  // (none past the rows that there are)
  if (context[b] <= 0) n = 0;
  n = n < 64 * N ? n : 64 * N;
  int64_t d[N], t[N];
  int p[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = 64 * k + lane;
    const bool in = i < n;
    d[k] = in ? draft[q0 + i] : 0;
    t[k] = in ? target[q0 + i] : 0;
    p[k] = in ? parents[q0 + i] : -1;
    if (p[k] >= i) p[k] = -1;
  }
  int count = 0, mine = -1;
  int64_t want = -1;
  for (int cur = n > 0 ? 0 : -1; cur >= 0;) {  // at most max_depth rounds
    if (lane == count) mine = cur;
    ++count;
    int64_t w = t[0];
#pragma unroll
    for (int k = 1; k < N; ++k)
      if (cur >> 6 == k) w = t[k];
    want = __shfl(w, cur & 63, 64);
    if (count == max_depth) break;
    int found = -1;
#pragma unroll
    for (int k = N - 1; k >= 0; --k) {
      const uint64_t on = __ballot(p[k] == cur && d[k] == want);
      if (on) found = 64 * k + __builtin_ctzll(on);
    }
    cur = found;  // a later node than cur
  }
  if (lane < max_depth) path[static_cast<int64_t>(b) * max_depth + lane] = mine;
  if (lane == 0) {
    accepted[b] = count;
    next[b] = want;
    if (pending != nullptr && count > 0) pending[b] = want;
    len_out[b] = L + count;
  }
}

}  // namespace wkv

using namespace wkv;

extern "C" int wkv_extend_tables_limited(int32_t *block_table, int64_t bt_stride, int32_t max_blocks_per_seq,
                                         const int32_t *held_blocks, const int32_t *seq_lens, const int32_t *new_lens,
                                         int32_t batch, int32_t block_size, const int32_t *free_blocks,
                                         int32_t num_free, const int32_t *taken, int32_t max_tokens,
                                         int32_t max_seq_len, const int32_t *parents, int32_t mask_words,
                                         int32_t *held_out, int32_t *taken_out, int32_t *context_lens,
                                         int32_t *cu_seqlens_q, int64_t *slot_mapping, int64_t *positions,
                                         int64_t *tree_mask, int32_t *refused, void *stream) {
  WKV_CHECK_ARG(batch > 0 && batch <= WKV_STEP_MAX_BATCH, "batch must be in [1, %d] (got %d)", WKV_STEP_MAX_BATCH, batch);
  WKV_CHECK_ARG(block_size > 0, "block_size must be positive (got %d)", block_size);
  WKV_CHECK_ARG(max_tokens >= 0 && max_tokens < INT32_MAX - 1024, "max_tokens must be in [0, 2^31 - 1025)");
  WKV_CHECK_ARG(max_seq_len >= 0, "max_seq_len must be >= 0 (got %d)", max_seq_len);
  WKV_CHECK_ARG(num_free >= 0 && num_free < INT32_MAX - 1, "num_free must be in [0, 2^31 - 2)");
  WKV_CHECK_ARG(block_table != nullptr && max_blocks_per_seq > 0 && bt_stride >= max_blocks_per_seq,
                "bad block table geometry");
  WKV_CHECK_ARG(held_blocks && seq_lens && new_lens && taken && held_out && taken_out && context_lens && cu_seqlens_q &&
                    refused && (free_blocks || num_free == 0) && ((slot_mapping && positions) || max_tokens == 0),
                "an input or output is NULL");
  WKV_CHECK_ARG(mask_words >= 0 && mask_words <= WKV_TREE_MAX_WORDS, "mask_words must be in [0, %d] (got %d)",
                WKV_TREE_MAX_WORDS, mask_words);
  WKV_CHECK_ARG(mask_words == 0 || max_tokens == 0 || (parents != nullptr && tree_mask != nullptr),
                "a tree needs parents and tree_mask");
  WKV_CHECK_ARG(context_lens != seq_lens && context_lens != new_lens && context_lens != held_blocks,
                "context_lens must not be one of the inputs");
  const TablesArgs a{block_table, bt_stride, max_blocks_per_seq, held_blocks, seq_lens, new_lens, free_blocks, taken,
                     num_free, batch, block_size, max_tokens, parents, mask_words, max_seq_len, held_out, taken_out,
                     context_lens, cu_seqlens_q, refused, slot_mapping, positions, tree_mask};
  auto s = static_cast<hipStream_t>(stream);
  if (max_tokens <= kTablesOwnRows) {
    tables_plan_kernel<true><<<1, kTablesThreads, 0, s>>>(a);
  } else {
    tables_plan_kernel<false><<<1, kTablesThreads, 0, s>>>(a);
    tables_rows_kernel<<<static_cast<unsigned>((static_cast<int64_t>(max_tokens) + 255) / 256), 256, 0, s>>>(a);
  }
  WKV_CHECK_LAUNCH("extend tables");
  return WKV_OK;
}

extern "C" int wkv_extend_tables(int32_t *block_table, int64_t bt_stride, int32_t max_blocks_per_seq,
                                 const int32_t *held_blocks, const int32_t *seq_lens, const int32_t *new_lens,
                                 int32_t batch, int32_t block_size, const int32_t *free_blocks, int32_t num_free,
                                 const int32_t *taken, int32_t max_tokens, const int32_t *parents, int32_t mask_words,
                                 int32_t *held_out, int32_t *taken_out, int32_t *context_lens, int32_t *cu_seqlens_q,
                                 int64_t *slot_mapping, int64_t *positions, int64_t *tree_mask, int32_t *refused,
                                 void *stream) {
  return wkv_extend_tables_limited(block_table, bt_stride, max_blocks_per_seq, held_blocks, seq_lens, new_lens, batch,
                                   block_size, free_blocks, num_free, taken, max_tokens, INT32_MAX, parents, mask_words,
                                   held_out, taken_out, context_lens, cu_seqlens_q, slot_mapping, positions, tree_mask,
                                   refused, stream);
}

extern "C" int wkv_accept_tree_pending(const int64_t *draft_tokens, const int32_t *parents,
                                       const int64_t *target_tokens, int64_t num_tokens, const int32_t *cu_seqlens_q,
                                       const int32_t *seq_lens, const int32_t *context_lens, int32_t batch,
                                       int32_t max_depth, int32_t *accepted, int32_t *path, int64_t *next_tokens,
                                       int32_t *seq_lens_out, int64_t *pending, void *stream) {
  WKV_CHECK_ARG(batch >= 0, "batch must be >= 0 (got %d)", batch);
  WKV_CHECK_ARG(max_depth > 0 && max_depth <= WKV_TREE_MAX_DEPTH, "max_depth must be in [1, %d] (got %d)",
                WKV_TREE_MAX_DEPTH, max_depth);
  WKV_CHECK_ARG(num_tokens >= 0 && num_tokens <= INT32_MAX, "num_tokens must be in [0, 2^31) (got %lld)",
                (long long)num_tokens);
  if (batch == 0) return WKV_OK;
  WKV_CHECK_ARG(((draft_tokens && parents && target_tokens) || num_tokens == 0) && cu_seqlens_q && seq_lens &&
                    context_lens && accepted && path && next_tokens && seq_lens_out,
                "an input or output is NULL");
  WKV_CHECK_ARG(pending != next_tokens, "pending must not be next_tokens");
  accept_tree_kernel<<<static_cast<unsigned>((batch + 3) / 4), 256, 0, static_cast<hipStream_t>(stream)>>>(
      draft_tokens, parents, target_tokens, static_cast<int>(num_tokens), cu_seqlens_q, seq_lens, context_lens, batch,
      max_depth, accepted, path, next_tokens, seq_lens_out, pending);
  WKV_CHECK_LAUNCH("accept tree");
  return WKV_OK;
}

extern "C" int wkv_accept_tree(const int64_t *draft_tokens, const int32_t *parents, const int64_t *target_tokens,
                               int64_t num_tokens, const int32_t *cu_seqlens_q, const int32_t *seq_lens,
                               const int32_t *context_lens, int32_t batch, int32_t max_depth, int32_t *accepted,
                               int32_t *path, int64_t *next_tokens, int32_t *seq_lens_out, void *stream) {
  return wkv_accept_tree_pending(draft_tokens, parents, target_tokens, num_tokens, cu_seqlens_q, seq_lens, context_lens,
                                 batch, max_depth, accepted, path, next_tokens, seq_lens_out, nullptr, stream);
}
