// Attention of sequences that share a prefix: token t of sequence b sees its group's prefix rows and its own rows up to its own.
#pragma once
#include "lane_rows.h"

namespace ajq {

struct SharedAttention {
  const void *q, *prefix_keys, *prefix_values, *keys, *values;
  const long long *prefix_lengths, *rows, *counts, *offset;
  uint16_t* out;
  long long prefix_group, prefix_head, cache_batch, cache_head;
  int groups, batch, tokens, heads, kv_heads, prefix_cap, max_len;
  float scale2;   // log2(e) / sqrt(dim)
};

__device__ __forceinline__ int held(long long n, int most) { return (int)min(max(n, 0ll), (long long)most); }

// A wave a query: four teams of sixteen lanes take rows in turn, the prefix's and then the sequence's own.
template <typename QT, typename CacheT, int HD>
__global__ __launch_bounds__(256) void shared_attention_plain_kernel(SharedAttention a) {
  using LD = LaneDims<float, HD>;
  constexpr int DPL = LD::DPL;
  const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);   // (b, h, t)
  if (id >= (long long)a.batch * a.heads * a.tokens) return;
  const int t = (int)(id % a.tokens), h = (int)(id / a.tokens % a.heads), b = (int)(id / a.tokens / a.heads);
  const int lane = threadIdx.x & 63, team = lane >> 4, c = lane & 15, d0 = LD::per_lane * c;
  const int hk = h / (a.heads / a.kv_heads), g = b / (a.batch / a.groups);
  const bool there = a.counts == nullptr || t < a.counts[b];
  const int before = there ? held(a.prefix_lengths[g], a.prefix_cap) : 0;
  const int own = there ? held(a.rows[b] + (a.offset ? *a.offset : 0ll) + t + 1, a.max_len) : 0;
  const KvRow<DPL> q = load_lane<HD>(reinterpret_cast<const QT*>(a.q) + (size_t)id * HD + d0);
  float m = -INFINITY, l = 0.f, acc[DPL] = {};
  auto walk = [&](const CacheT* keys, const CacheT* values, int rows) {
    for (int i = team; i < rows; i += 4) {
      const KvRow<DPL> k = load_lane<HD>(keys + (size_t)i * HD + d0), v = load_lane<HD>(values + (size_t)i * HD + d0);
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < DPL; ++j) s += q.v[j] * k.v[j];
      s = team_sum16(s) * a.scale2;
      const float m_new = fmaxf(m, s), corr = exp2_hw(m - m_new), w = exp2_hw(s - m_new);
      l = l * corr + w;
#pragma unroll
      for (int j = 0; j < DPL; ++j) acc[j] = acc[j] * corr + w * v.v[j];
      m = m_new;
    }
  };
  const size_t at = (size_t)g * a.prefix_group + (size_t)hk * a.prefix_head, mine = (size_t)b * a.cache_batch + (size_t)hk * a.cache_head;
  walk(reinterpret_cast<const CacheT*>(a.prefix_keys) + at, reinterpret_cast<const CacheT*>(a.prefix_values) + at, before);
  walk(reinterpret_cast<const CacheT*>(a.keys) + mine, reinterpret_cast<const CacheT*>(a.values) + mine, own);
#pragma unroll
  for (int off = 16; off <= 32; off <<= 1) {
    const float mo = __shfl_xor(m, off), lo = __shfl_xor(l, off), top = fmaxf(m, mo);
    const float cm = m == -INFINITY ? 0.f : exp2_hw(m - top), co = mo == -INFINITY ? 0.f : exp2_hw(mo - top);
    l = l * cm + lo * co;
#pragma unroll
    for (int j = 0; j < DPL; ++j) acc[j] = acc[j] * cm + __shfl_xor(acc[j], off) * co;
    m = top;
  }
  if (team != 0) return;
  KvRow<DPL> o{};
  if (l != 0.f) {
#pragma unroll
    for (int j = 0; j < DPL; ++j) o.v[j] = acc[j] / l;
  }
  store_lane<HD>(a.out + ((size_t)b * a.tokens + t) * ((size_t)a.heads * HD) + (size_t)h * HD + d0, o);
}

}  // namespace ajq
