// Rows of a key / value cache dealt to teams of sixteen lanes, and what else small kernels share.
#pragma once
#include "ajq_common.h"

namespace ajq {

// Which HD / 16 of a row's dimensions lane c of a team holds (DPL of them: 8, 4 or 2), and how it fetches them.
// 8 per lane, bf16 rows (256 B): 8c .. 8c+7, one 128-bit load.  8 per lane, fp32 rows (512 B): 4c .. 4c+3
// and 64+4c .. 64+4c+3, so each of a team's two 128-bit loads covers 256 contiguous bytes.  4 per lane:
// 4c .. 4c+3, one 128-bit (fp32) or 64-bit (bf16) load.  2 per lane: 2c, 2c+1, one 64-bit or 32-bit load.
template <typename CacheT, int HD> struct LaneDims {
  static_assert(HD == 128 || HD == 64 || HD == 32, "head_dim 128, 64 or 32");
  static constexpr int DPL = HD / 16;
  static constexpr bool split = sizeof(CacheT) == 4 && DPL == 8;
  static constexpr int per_lane = split ? 4 : DPL;   // the lane's first dimension = per_lane * c
  static constexpr int second = split ? 64 : 4;      // DPL == 8: its second four start this many dimensions later
  __device__ static __forceinline__ int dim(int c, int i) { return per_lane * c + (i < 4 ? i : second + i - 4); }
};
template <int DPL> struct KvRow {
  float v[DPL];
};
template <bool kStream, typename T>
__device__ __forceinline__ T load_kv(const T* p) {
  if constexpr (kStream) return __builtin_nontemporal_load(p);
  return *p;
}
__device__ __forceinline__ void widen2(uint32_t w, float& lo, float& hi) {  // two bf16 -> two fp32
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xFFFF0000u);
}
// A row of the cache as loaded (the lane's dimensions; p: the first of them) and widened to fp32 when it is used, so that a row
// on its way from memory costs no more registers than its bytes.
template <typename CacheT, int HD> struct RawRow {
  static constexpr int words = (HD / 16) * (int)sizeof(CacheT) / 4;  // 8, 4, 2 (fp32) or 4, 2, 1 (bf16)
  uint32_t w[words];
};
template <bool kStream, int HD, typename CacheT>
__device__ __forceinline__ RawRow<CacheT, HD> load_raw(const CacheT* p) {
  constexpr int words = RawRow<CacheT, HD>::words;
  RawRow<CacheT, HD> r;
  if constexpr (words >= 4) {
#pragma unroll
    for (int h = 0; h < words / 4; ++h) {
      const u32x4_t a = load_kv<kStream>(reinterpret_cast<const u32x4_t*>(p + h * LaneDims<CacheT, HD>::second));
      r.w[4 * h] = a.x; r.w[4 * h + 1] = a.y; r.w[4 * h + 2] = a.z; r.w[4 * h + 3] = a.w;
    }
  } else if constexpr (words == 2) {
    const u32x2_t a = load_kv<kStream>(reinterpret_cast<const u32x2_t*>(p));
    r.w[0] = a.x; r.w[1] = a.y;
  } else {
    r.w[0] = load_kv<kStream>(reinterpret_cast<const uint32_t*>(p));
  }
  return r;
}
template <typename CacheT, int HD>
__device__ __forceinline__ KvRow<HD / 16> widen_row(const RawRow<CacheT, HD>& raw) {
  KvRow<HD / 16> r;
#pragma unroll
  for (int i = 0; i < RawRow<CacheT, HD>::words; ++i) {
    if constexpr (sizeof(CacheT) == 4) r.v[i] = __uint_as_float(raw.w[i]);
    else widen2(raw.w[i], r.v[2 * i], r.v[2 * i + 1]);
  }
  return r;
}
// 2^x by the hardware instruction (1 ulp); the softmax below keeps its running maximum and
// scores in the base-2 domain, scores pre-multiplied by log2(e)
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float kLog2e = 1.4426950408889634f;

// a lane's DPL components at p (its first one), as LaneDims<float, HD> places them
template <int HD>
__device__ __forceinline__ KvRow<HD / 16> load_lane(const float* p) {
  using LD = LaneDims<float, HD>;
  KvRow<HD / 16> r;
  if constexpr (LD::DPL == 2) {
    const float2 a = *reinterpret_cast<const float2*>(p);
    r.v[0] = a.x; r.v[1] = a.y;
  } else {
    const float4 a = *reinterpret_cast<const float4*>(p);
    r.v[0] = a.x; r.v[1] = a.y; r.v[2] = a.z; r.v[3] = a.w;
    if constexpr (LD::DPL == 8) {
      const float4 b = *reinterpret_cast<const float4*>(p + LD::second);
      r.v[4] = b.x; r.v[5] = b.y; r.v[6] = b.z; r.v[7] = b.w;
    }
  }
  return r;
}
template <int HD>
__device__ __forceinline__ KvRow<HD / 16> load_lane(const uint16_t* p) {
  using LD = LaneDims<float, HD>;
  KvRow<HD / 16> r;
  if constexpr (LD::DPL == 2) {
    widen2(*reinterpret_cast<const uint32_t*>(p), r.v[0], r.v[1]);
  } else {
    const u32x2_t a = *reinterpret_cast<const u32x2_t*>(p);
    widen2(a.x, r.v[0], r.v[1]);
    widen2(a.y, r.v[2], r.v[3]);
    if constexpr (LD::DPL == 8) {
      const u32x2_t b = *reinterpret_cast<const u32x2_t*>(p + LD::second);
      widen2(b.x, r.v[4], r.v[5]);
      widen2(b.y, r.v[6], r.v[7]);
    }
  }
  return r;
}
template <int HD>
__device__ __forceinline__ void store_lane(float* p, const KvRow<HD / 16>& r) {
  using LD = LaneDims<float, HD>;
  if constexpr (LD::DPL == 2) {
    *reinterpret_cast<float2*>(p) = float2{r.v[0], r.v[1]};
  } else {
    *reinterpret_cast<float4*>(p) = float4{r.v[0], r.v[1], r.v[2], r.v[3]};
    if constexpr (LD::DPL == 8) *reinterpret_cast<float4*>(p + LD::second) = float4{r.v[4], r.v[5], r.v[6], r.v[7]};
  }
}
template <int HD>
__device__ __forceinline__ void store_lane(uint16_t* p, const KvRow<HD / 16>& r) {
  using LD = LaneDims<float, HD>;
  if constexpr (LD::DPL == 2) {
    *reinterpret_cast<uint32_t*>(p) = pack2_bf16(r.v[0], r.v[1]);
  } else {
    *reinterpret_cast<u32x2_t*>(p) = u32x2_t{pack2_bf16(r.v[0], r.v[1]), pack2_bf16(r.v[2], r.v[3])};
    if constexpr (LD::DPL == 8) *reinterpret_cast<u32x2_t*>(p + LD::second) = u32x2_t{pack2_bf16(r.v[4], r.v[5]), pack2_bf16(r.v[6], r.v[7])};
  }
}

// Division by a number that the host knows: the product with 2^32 / d rounded down is the quotient or one less for every 32-bit n.  (A division of
// its own is some forty instructions, at the start of a kernel that runs for a few microseconds a third of its instructions.)
struct Divide {
  uint32_t d, m;
};
__host__ inline Divide divide_by(long long d) { return Divide{(uint32_t)d, (uint32_t)((d > 1 ? (1ll << 32) / d : 0xFFFFFFFFll))}; }
__device__ __forceinline__ int divide(int n, const Divide& by, int& rest) {
  int q = (int)__umulhi((uint32_t)n, by.m);
  rest = n - q * (int)by.d;
  if (rest >= (int)by.d) {
    rest -= (int)by.d;
    ++q;
  }
  return q;
}

}  // namespace ajq
