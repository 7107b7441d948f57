// Queries and keys of a projection's output: RMS norm over each head, rotation of its pairs, keys and values into the caches, for sequences
// at positions of their own.
//
//   y = x / sqrt(mean(x^2) + eps) * gain;  (y[2i], y[2i+1]) -> (y[2i] c_i - y[2i+1] s_i, y[2i] s_i + y[2i+1] c_i)
//
// Sixteen lanes hold a head (dim / 16 components each, in the places LaneDims gives them), so the sum of squares is four DPP adds and
// a pair never leaves its lane.  Everything is read once and written once.
#pragma once
#include "lane_rows.h"

namespace ajq {

struct NormRope {
  const void* qkv;
  const float *cosine, *sine, *q_gain, *k_gain;
  const long long *rows, *positions, *counts, *offset;
  void *keys, *values, *q;
  long long ld, cache_batch, cache_head;
  int tokens, heads, kv_heads, max_len, table_rows;
  float eps;
};

// Workgroup (m, y): token m, heads 16 U y .. of its heads + 2 kv_heads, U a team of sixteen lanes, all requested before any is used.
template <typename InT, typename QT, typename CacheT, int HD, int U>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRope a) {
  using LD = LaneDims<float, HD>;
  constexpr int DPL = LD::DPL;
  const int m = blockIdx.x, b = m / a.tokens, t = m % a.tokens;
  const int team = threadIdx.x >> 4, c = threadIdx.x & 15, d0 = LD::per_lane * c;
  const int all = a.heads + 2 * a.kv_heads, first = blockIdx.y * (16 * U) + team;
  const InT* row = reinterpret_cast<const InT*>(a.qkv) + (size_t)m * a.ld + d0;
  KvRow<DPL> x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) x[u] = load_lane<HD>(row + (size_t)min(first + 16 * u, all - 1) * HD);
  const long long off = a.offset ? *a.offset : 0ll;
  const long long at = a.rows[b] + off + t;
  const long long p = min(max((a.positions ? a.positions[b] + off : a.rows[b] + off) + t, 0ll), (long long)a.table_rows - 1);
  const bool there = a.counts == nullptr || t < a.counts[b];
  float cs[DPL / 2], sn[DPL / 2];
#pragma unroll
  for (int i = 0; i < DPL / 2; ++i) {
    const size_t pair = (size_t)p * (HD / 2) + LD::dim(c, 2 * i) / 2;
    cs[i] = a.cosine[pair];
    sn[i] = a.sine[pair];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int head = first + 16 * u;
    if (head >= all) break;
    const bool query = head < a.heads, value = head >= a.heads + a.kv_heads;
    const float* gain = value ? nullptr : query ? a.q_gain : a.k_gain;
    if (gain) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < DPL; ++i) ss += x[u].v[i] * x[u].v[i];
      const Divisor by_rms(sqrtf(team_sum16(ss) / (float)HD + a.eps));
      const KvRow<DPL> g = load_lane<HD>(gain + d0);
#pragma unroll
      for (int i = 0; i < DPL; ++i) x[u].v[i] = by_rms.divide(x[u].v[i]) * g.v[i];
    }
    if (!value) {
#pragma unroll
      for (int i = 0; i < DPL / 2; ++i) {
        const float e = x[u].v[2 * i], o = x[u].v[2 * i + 1];
        x[u].v[2 * i] = e * cs[i] - o * sn[i];
        x[u].v[2 * i + 1] = e * sn[i] + o * cs[i];
      }
    }
    if (query) {
      if (!there) x[u] = KvRow<DPL>{};
      store_lane<HD>(reinterpret_cast<QT*>(a.q) + (((size_t)b * a.heads + head) * a.tokens + t) * HD + d0, x[u]);
    } else if (there && at >= 0 && at < a.max_len) {
      const int g = value ? head - a.heads - a.kv_heads : head - a.heads;
      CacheT* cache = reinterpret_cast<CacheT*>(value ? a.values : a.keys);
      store_lane<HD>(cache + (size_t)b * a.cache_batch + (size_t)g * a.cache_head + (size_t)at * HD + d0, x[u]);
    }
  }
}

}  // namespace ajq
