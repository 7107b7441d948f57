// Attention of a tree of drafted tokens over a cache: each sees the committed rows and, of the tokens' own, those whose bits its mask has.
//
//   out[b, t, h] = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c q . k_j - m),  c = log2(e) / sqrt(HD)
#pragma once
#include "lane_rows.h"

namespace ajq {

struct TreeAttention {
  const void *q, *keys, *values;
  const uint32_t* masks;
  const long long *rows, *counts, *offset;
  uint16_t* out;
  long long cache_batch, cache_head, mask_batch, mask_token;
  int batch, tokens, heads, kv_heads, max_len;
  float scale2;
};

// A wave a query, a team of sixteen lanes a row.
template <int HD, typename QT, typename CacheT>
__global__ __launch_bounds__(64) void tree_attention_kernel(TreeAttention a) {
  using LD = LaneDims<float, HD>;
  constexpr int DPL = LD::DPL;
  const int team = threadIdx.x >> 4, c = threadIdx.x & 15, d0 = LD::per_lane * c;
  const int t = blockIdx.x, h = blockIdx.y, b = blockIdx.z, g = h / (a.heads / a.kv_heads);
  const long long before = min(max(a.rows[b] + (a.offset ? *a.offset : 0ll), -(1ll << 30)), 1ll << 30);
  const int there = a.counts ? (int)min(max(a.counts[b], 0ll), (long long)a.tokens) : a.tokens;
  const int rows = (int)min(max(before + there, 0ll), (long long)a.max_len);
  const KvRow<DPL> q = load_lane<HD>(reinterpret_cast<const QT*>(a.q) + (((size_t)b * a.heads + h) * a.tokens + t) * HD + d0);
  const size_t at = (size_t)b * a.cache_batch + (size_t)g * a.cache_head + d0;
  const CacheT *keys = reinterpret_cast<const CacheT*>(a.keys) + at, *values = reinterpret_cast<const CacheT*>(a.values) + at;
  const uint32_t* mask = a.masks + b * a.mask_batch + t * a.mask_token;
  float m = -INFINITY, l = 0.f;
  KvRow<DPL> o = {};
  for (int j = team; t < there && j < rows; j += 4) {
    const long long node = j - before;
    if (node >= 0 && !(mask[node >> 5] >> (node & 31) & 1)) continue;   // (a team's lanes together)
    const KvRow<DPL> k = load_lane<HD>(keys + (size_t)j * HD), v = load_lane<HD>(values + (size_t)j * HD);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) dot += q.v[i] * k.v[i];
    const float x = team_sum16(dot) * a.scale2, top = fmaxf(m, x);
    const float old = m == -INFINITY ? 0.f : exp2_hw(m - top), p = exp2_hw(x - top);
    m = top;
    l = l * old + p;
#pragma unroll
    for (int i = 0; i < DPL; ++i) o.v[i] = o.v[i] * old + p * v.v[i];
  }
  const float top = quad_max(m), weight = m == -INFINITY ? 0.f : exp2_hw(m - top);
  l = quad_sum(l * weight);
#pragma unroll
  for (int i = 0; i < DPL; ++i) {
    const float x = quad_sum(o.v[i] * weight);
    o.v[i] = l != 0.f ? x / l : 0.f;
  }
  if (team == 0) store_lane<HD>(a.out + (((size_t)b * a.tokens + t) * a.heads + h) * HD + d0, o);
}

}  // namespace ajq
