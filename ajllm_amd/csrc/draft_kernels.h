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

// ---- rows that stay.  A workgroup has a head's keys or values to itself and takes its list in pieces of blockDim / lanes-a-row rows, 16 bytes a
// lane.  A piece is loaded, then all wait, then it is stored: what a store overwrites (rows ahead of the piece's end) no later piece reads, since the
// numbers ascend.
struct KeepRows {
  void *keys, *values;
  const long long *rows, *index, *counts, *offset;
  long long cache_layer, cache_batch, cache_head, index_ld;   // (elements)
  int batch, kv_heads, max_len, width, row_bytes, element;
};
__global__ __launch_bounds__(1024) void keep_rows_kernel(KeepRows a) {
  __shared__ int broken;   // the first place of the piece whose number does not ascend
  const int lanes = a.row_bytes / 16, row = threadIdx.x / lanes, lane = threadIdx.x % lanes, each = blockDim.x / lanes;
  const int which = blockIdx.x & 1;
  int id = blockIdx.x >> 1;
  const int head = id % a.kv_heads;
  id /= a.kv_heads;
  const int b = id % a.batch, layer = id / a.batch;
  char* cache = reinterpret_cast<char*>(which ? a.values : a.keys) +
                (size_t)(layer * a.cache_layer + b * a.cache_batch + head * a.cache_head) * a.element + 16 * lane;
  const long long first = a.rows[b] + (a.offset ? *a.offset : 0ll);
  if (first < 0 || first >= a.max_len) return;
  const int room = a.max_len - (int)first;
  cache += first * a.row_bytes;
  const int count = min(a.counts ? (int)min(max(a.counts[b], 0ll), (long long)a.width) : a.width, room);
  const long long* index = a.index + b * a.index_ld;
  for (int begin = 0; begin < count; begin += each) {
    const int i = begin + row;
    if (threadIdx.x == 0) broken = count;
    __syncthreads();
    long long from = -1;
    u32x4_t x = {};
    if (i < count) {
      from = index[i];
      if (from < 0 || from >= room || (i > 0 && from <= index[i - 1])) atomicMin(&broken, i);
      else if (from != i) x = *reinterpret_cast<const u32x4_t*>(cache + from * a.row_bytes);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (what another wave overwrites next has been read)
    __syncthreads();
    const int last = broken;
    __syncthreads();
    if (i < last && from != i) *reinterpret_cast<u32x4_t*>(cache + (size_t)i * a.row_bytes) = x;
    if (last < count) break;
  }
}

}  // namespace ajq
