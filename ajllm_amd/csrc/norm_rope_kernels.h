// Queries and keys of a projection's output: RMS norm over each head, rotation of its pairs, keys and values into the caches, for sequences
// at positions of their own.
//
//   y = x / sqrt(mean(x^2) + eps) * gain;  (y[2i], y[2i+1]) -> (y[2i] c_i - y[2i+1] s_i, y[2i] s_i + y[2i+1] c_i)
//
// Sixteen lanes hold a head (dim / 16 components each, in the places LaneDims gives them), so the sum of squares is four DPP adds and
// a pair never leaves its lane.  Everything is read once and written once, which is what bounds it: 16 prompts of 333 tokens (32 + 16 heads of 128, fp32 in,
// bf16 out, 160 MB) 28.2 to 30.0 us = 5.3 to 5.7 TB/s; a token of each of 96 sequences 3.3 us, of 8 2.8, of which a launch takes 2.6.
#pragma once
#include "lane_rows.h"

namespace ajq {

struct NormRope {
  const void* qkv;
  const float *cosine, *sine, *q_gain, *k_gain;
  const long long *rows, *positions, *counts, *offset, *depths;
  void *keys, *values, *q;
  long long ld, cache_batch, cache_head, depths_ld;
  int tokens, heads, kv_heads, max_len, table_rows;
  float eps;
  Divide by_tokens;
};

// Workgroup (m, y): token m, heads 16 U y .. of its heads + 2 kv_heads, U a team of sixteen lanes, all requested before any is used.  A single
// token a sequence asks for its components ahead of anything it reads on the device: a launch's round trips are all it takes.  Of several
// (kMany) those that are not there ask for nothing, and what is read and written once goes past L2.
template <bool kMany, typename T>
__device__ __forceinline__ T load_once(const T* p) {
  if constexpr (kMany) return __builtin_nontemporal_load(p);
  return *p;
}
template <bool kMany, int HD>
__device__ __forceinline__ KvRow<HD / 16> ask_lane(const float* p) {
  using LD = LaneDims<float, HD>;
  KvRow<HD / 16> r;
  if constexpr (LD::DPL == 2) {
    const u32x2_t a = load_once<kMany>(reinterpret_cast<const u32x2_t*>(p));
    r.v[0] = __uint_as_float(a.x); r.v[1] = __uint_as_float(a.y);
  } else {
    const f32x4_t a = load_once<kMany>(reinterpret_cast<const f32x4_t*>(p));
    r.v[0] = a.x; r.v[1] = a.y; r.v[2] = a.z; r.v[3] = a.w;
    if constexpr (LD::DPL == 8) {
      const f32x4_t b = load_once<kMany>(reinterpret_cast<const f32x4_t*>(p + LD::second));
      r.v[4] = b.x; r.v[5] = b.y; r.v[6] = b.z; r.v[7] = b.w;
    }
  }
  return r;
}
template <bool kMany, int HD>
__device__ __forceinline__ KvRow<HD / 16> ask_lane(const uint16_t* p) { return load_lane<HD>(p); }

template <typename InT, typename QT, typename CacheT, int HD, int U, bool kMany>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRope a) {
  using LD = LaneDims<float, HD>;
  constexpr int DPL = LD::DPL;
  int t = 0;
  const int m = blockIdx.x, b = kMany ? divide(m, a.by_tokens, t) : m;
  const int team = threadIdx.x >> 4, c = threadIdx.x & 15, d0 = LD::per_lane * c;
  const int all = a.heads + 2 * a.kv_heads, first = blockIdx.y * (16 * U) + team;
  const InT* row = reinterpret_cast<const InT*>(a.qkv) + (size_t)m * a.ld + d0;
  const bool there = a.counts == nullptr || t < a.counts[b];
  KvRow<DPL> x[U] = {};
  if (!kMany || there) {
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = ask_lane<kMany, HD>(row + (size_t)min(first + 16 * u, all - 1) * HD);
  }
  const long long off = a.offset ? *a.offset : 0ll;
  const long long at = a.rows[b] + off + t;
  const long long p = min(max((a.positions ? a.positions[b] + off : a.rows[b] + off) + (a.depths ? a.depths[b * a.depths_ld + t] : t), 0ll), (long long)a.table_rows - 1);
  float cs[DPL / 2], sn[DPL / 2];
#pragma unroll
  for (int i = 0; i < DPL / 2; ++i) {
    const size_t pair = (size_t)p * (HD / 2) + LD::dim(c, 2 * i) / 2;
    cs[i] = a.cosine[pair];
    sn[i] = a.sine[pair];
  }
  // (both gains, whichever a head takes: they come with the components)
  KvRow<DPL> gain[2] = {};
  if (a.q_gain) gain[0] = load_lane<HD>(a.q_gain + d0);
  if (a.k_gain) gain[1] = load_lane<HD>(a.k_gain + d0);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int head = first + 16 * u;
    if (head >= all) break;
    const bool query = head < a.heads, value = head >= a.heads + a.kv_heads;
    if (!value && (query ? a.q_gain : a.k_gain)) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < DPL; ++i) ss += x[u].v[i] * x[u].v[i];
      float mean = team_sum16(ss) / (float)HD + a.eps;
      if (!(mean >= 0x1p-100f && mean <= 0x1.fffffep127f)) {
        // squares past what fp32 holds (components above 1.6e18), or lost at its lower end (no epsilon, components below 1e-15): the same of x times a power of two
        const float by = mean > 1.f ? 0x1p-100f : 0x1p100f;
        ss = 0.f;
#pragma unroll
        for (int i = 0; i < DPL; ++i) {
          x[u].v[i] *= by;
          ss += x[u].v[i] * x[u].v[i];
        }
        mean = team_sum16(ss) / (float)HD + a.eps * by * by;
      }
      const Divisor by_rms(sqrtf(mean));
#pragma unroll
      for (int i = 0; i < DPL; ++i) x[u].v[i] = by_rms.divide(x[u].v[i]) * (query ? gain[0].v[i] : gain[1].v[i]);
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
