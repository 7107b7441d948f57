// The small operators of checking drafted tokens: the path that the model's choices take through a tree, and the rows of it that stay.
#pragma once
#include "lane_rows.h"

namespace ajq {

// ---- the path.  Every node looks whether it guesses the choice behind its parent, and the first child that does becomes its parent's next; then one
// lane walks from the root through LDS.  (Whole numbers and a minimum: no result depends on the order of the atomics.)
constexpr int kMostNodes = 4096, kFollowThreads = 256;
struct FollowDrafts {
  const long long *tokens, *parents, *choices, *counts;
  long long *path, *accepted, *chosen;
  long long tokens_ld, parents_ld, choices_ld, choices_step;
  int nodes;
};
__global__ __launch_bounds__(kFollowThreads) void follow_drafts_kernel(FollowDrafts a) {
  __shared__ int next[kMostNodes], path[kMostNodes];
  __shared__ int length;
  const int b = blockIdx.x;
  const int there = a.counts ? (int)min(max(a.counts[b], 0ll), (long long)a.nodes) : a.nodes;
  const long long *tokens = a.tokens + b * a.tokens_ld, *parents = a.parents + b * a.parents_ld, *choices = a.choices + b * a.choices_ld;
  for (int t = threadIdx.x; t < a.nodes; t += blockDim.x) next[t] = a.nodes;
  __syncthreads();
  for (int t = threadIdx.x; t < there; t += blockDim.x) {
    const long long up = parents[t];
    if (t > 0 && up >= 0 && up < t && tokens[t] == choices[up * a.choices_step]) atomicMin(&next[up], t);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = 0;
    for (int at = 0; at < there; at = next[at]) path[n++] = at;   // (ascending: n stays below the nodes)
    length = n;
    a.accepted[b] = n;
  }
  __syncthreads();
  for (int t = threadIdx.x; t < a.nodes; t += blockDim.x) {
    const bool on = t < length;
    a.path[(size_t)b * a.nodes + t] = on ? path[t] : -1;
    a.chosen[(size_t)b * a.nodes + t] = on ? choices[path[t] * a.choices_step] : -1;
  }
}

// ---- rows that stay.  A workgroup has a head's keys or values to itself, 16 bytes a lane.  What a store overwrites is a row ahead of the list's end at that point,
// which nothing behind it reads, since the numbers ascend: rows are loaded, then all wait, then they are stored.
struct KeepRows {
  void *keys, *values;
  const long long *rows, *index, *counts, *offset;
  long long cache_layer, cache_batch, cache_head, index_ld;   // (elements)
  int max_len, width, row_bytes, element, lanes;   // (lanes: 16 bytes each, of a row that a workgroup takes)
  Divide by_columns, by_heads, by_batch;            // (columns: parts of a row, a workgroup each)
};
struct KeptHead {
  char* cache;              // the lane's 16 bytes of the list's row 0
  const long long* index;
  int count, room;          // numbers of the list (0: none), rows from its row 0 on
};
__device__ __forceinline__ KeptHead kept_head(const KeepRows& a, int lane) {
  KeptHead h;
  int column, head, b;
  const int layer = divide(divide(divide((int)(blockIdx.x >> 1), a.by_columns, column), a.by_heads, head), a.by_batch, b);
  const long long first = a.rows[b] + (a.offset ? *a.offset : 0ll), count = a.counts ? a.counts[b] : a.width;
  const bool inside = first >= 0 && first < a.max_len;
  h.room = inside ? a.max_len - (int)first : 0;
  h.count = (int)min(max(count, 0ll), (long long)min(a.width, h.room));
  h.cache = reinterpret_cast<char*>(blockIdx.x & 1 ? a.values : a.keys) +
            (size_t)(layer * a.cache_layer + b * a.cache_batch + head * a.cache_head) * a.element + (inside ? first : 0) * a.row_bytes + 16 * (column * a.lanes + lane);
  h.index = a.index + b * a.index_ld;
  return h;
}

// Up to 64 numbers: each wave has them in its lanes, a vote says where they end, and one wait is enough for all rows.  A launch and two round trips, the list's and
// the rows': a path through 16 nodes in twelve layers of 8 x 16 heads of 128 (fp32, 20 MB read and written) 6.9 us (by pieces as below 8.5); 64 in 32
// layers of 32 x 8 heads (bf16, 215 MB) 37 us (42).  Eight rows a lane took 244 registers, and 14 us for the first.
constexpr int kShortList = 64;
template <int kMost>   // rows a lane
__global__ __launch_bounds__(256) void keep_path_kernel(KeepRows a) {
  const int row = threadIdx.x / a.lanes, each = 256 / a.lanes, wave_lane = threadIdx.x & 63;
  const KeptHead h = kept_head(a, threadIdx.x % a.lanes);
  const long long number = h.index[min(wave_lane, a.width - 1)], ahead = __shfl_up(number, 1);
  const bool on = wave_lane < h.count && number >= 0 && number < h.room && (wave_lane == 0 || number > ahead);
  const unsigned long long ends = __builtin_amdgcn_ballot_w64(!on);
  const int many = ends ? __builtin_ctzll(ends) : 64, from = (int)number;
  u32x4_t x[kMost] = {};
  bool moves[kMost];
#pragma unroll
  for (int p = 0; p < kMost; ++p) {
    const int i = p * each + row, source = __shfl(from, i & 63);
    moves[p] = i < many && source != i;
    if (moves[p]) x[p] = *reinterpret_cast<const u32x4_t*>(h.cache + (size_t)source * a.row_bytes);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (what another wave overwrites next has been read)
  __syncthreads();
#pragma unroll
  for (int p = 0; p < kMost; ++p)
    if (moves[p]) *reinterpret_cast<u32x4_t*>(h.cache + (size_t)(p * each + row) * a.row_bytes) = x[p];
}

// Longer ones in pieces of a row a lane.  The next piece's rows are on their way while one is stored: what is stored lies ahead of all of them.  Half of 8192 rows
// of 512 heads (bf16, 128), 2.15 GB read and written, 404 us = 5.3 TB/s (two rows a lane 405, four 411; 512 lanes and two rows 416).  Of 16 heads (fp32) 45 us with a
// quarter of a row a workgroup, 150 with whole ones.
__global__ __launch_bounds__(1024) void keep_rows_kernel(KeepRows a) {
  __shared__ int ends[2];   // of the piece: where it ends early (two in turn: the next piece's while this one's is read)
  const int row = threadIdx.x / a.lanes, each = 1024 / a.lanes;
  const KeptHead h = kept_head(a, threadIdx.x % a.lanes);
  if (threadIdx.x < 2) ends[threadIdx.x] = h.count;
  __syncthreads();
  // row i's source (i itself: it stays), and what is there
  auto fetch = [&](int i, int& source, int& end) __attribute__((always_inline)) {
    u32x4_t x = {};
    source = i;
    if (i >= h.count) return x;
    const long long number = h.index[i], ahead = i > 0 ? h.index[i - 1] : -1;
    if (number < 0 || number >= h.room || number <= ahead) {
      atomicMin(&end, i);
    } else {
      source = (int)number;
      if (source != i) x = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(h.cache + (size_t)source * a.row_bytes));
    }
    return x;
  };
  int source;
  u32x4_t x = fetch(row, source, ends[0]);
  for (int begin = 0, turn = 0; begin < h.count; begin += each, turn ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (what another wave overwrites next has been read)
    __syncthreads();
    const int end = ends[turn], i = begin + row;
    int next_source = i + each;
    u32x4_t next = {};
    if (end == h.count) next = fetch(i + each, next_source, ends[turn ^ 1]);
    if (i < end && source != i) __builtin_nontemporal_store(x, reinterpret_cast<u32x4_t*>(h.cache + (size_t)i * a.row_bytes));
    if (end < h.count) break;
    source = next_source;
    x = next;
  }
}

}  // namespace ajq
