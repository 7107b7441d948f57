// Attention of a tree of drafted tokens over a cache: each sees the committed rows and, of the tokens' own behind them, those whose bits its mask has.
//
//   out[b, t, h] = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c q . k_j - m),  c = log2(e) / sqrt(HD)
//
// All of a sequence's tokens see nearly the same rows, so that a key head's rows meet tokens * share queries as a matrix product's, by the ways of
// shared_attention.h: meet_few by tiles of 16 or 32 queries, meet_many by 64 or 128.  There the rows are one run, cut into parts where tiles are few; a block of
// 32 of them is seen by everybody, or (two or three at the end) by those queries whose bits say so: one shift of two mask words a query.
#pragma once
#include "shared_attention.h"

namespace ajq {

struct TreeAttention : SharedAttention {   // (the prefix's caches are the sequences' own; prefix_blocks, prefix_parts 0)
  const uint32_t* masks;
  long long mask_batch, mask_token;
  static constexpr bool kTree = true;
};
template <> struct SeenBits<TreeAttention> {
  const uint32_t* mask;
  uint32_t first;
  __device__ __forceinline__ void ask(const TreeAttention& a, int sequence, int token) {
    mask = a.masks + sequence * a.mask_batch + token * a.mask_token;
    first = mask[0];
  }
  __device__ __forceinline__ uint32_t word(const TreeAttention& a, int n) const {
    return n < 0 ? ~0u : n == 0 ? first : 32 * n < a.tokens ? mask[n] : 0u;
  }
  // bit i: own row at + i
  __device__ __forceinline__ uint32_t of(const TreeAttention& a, int at) const {
    const int n = at >> 5;
    return __builtin_amdgcn_alignbit(word(a, n + 1), word(a, n), (uint32_t)at & 31u);
  }
};

// A tile's queries and a part of the rows to a workgroup (kWhole: all rows, and what comes out is the result).
template <int HD, typename QT, typename CacheT, int RT, bool kWhole>
__global__ __launch_bounds__(256, sizeof(CacheT) == 4 && RT == 2 ? 1 : 2) void tree_attention_few_kernel(TreeAttention a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char shared_lds[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(pf_lds_char_t*)shared_lds;
  Meeting<CacheT> w;
  if (!find_meeting<CacheT, HD>(a, 16, 16 * RT, w)) return;
  meet_some<HD, QT, CacheT, RT, false, kWhole>(a, w, shared_lds, lds0);
}
template <int HD, typename QT, int U>
__global__ __launch_bounds__(256, 2) void tree_attention_walk_kernel(TreeAttention a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char shared_lds[];
  walk_own<HD, QT, U>(a, (uint32_t)(uintptr_t)(pf_lds_char_t*)shared_lds);
}

}  // namespace ajq
