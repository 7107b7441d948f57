// Log probabilities of given tokens, entropies, and the first tokens in the order of their logits.
//
//   log p_t = (x_t - m) - log s,   H = log s - u / s,   m = max x_v,   s = sum e^(x_v - m),   u = sum e^(x_v - m) (x_v - m)
#pragma once
#include "lane_rows.h"

namespace ajq {

constexpr int kMostTop = 64;
struct LogProbs {
  const void* logits;
  const long long* targets;
  float *log_probs, *entropy, *top_log_probs;
  long long *ranks, *top_ids;
  long long ld;
  int rows, vocab, top;
};

// The order of the tokens as whole numbers: larger logits first (NaN ahead of all, -0 as 0), then smaller ids.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t bits = __float_as_uint(x + 0.f);
  return x != x ? 0xFFFFFFFFu : bits ^ ((uint32_t)((int)bits >> 31) | 0x80000000u);
}
__device__ __forceinline__ unsigned long long key_of(float x, int id) { return (unsigned long long)order_of(x) << 32 | (uint32_t)~id; }
__device__ __forceinline__ float logit(const float* p) { return *p; }
__device__ __forceinline__ float logit(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }

// fn over a workgroup of 256 lanes; every lane gets the result
template <typename T, typename F>
__device__ __forceinline__ T over_group(T v, T* room, F&& fn) {
  __syncthreads();
  room[threadIdx.x] = v;
  for (int n = 128; n > 0; n >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < n) room[threadIdx.x] = fn(room[threadIdx.x], room[threadIdx.x + n]);
  }
  __syncthreads();
  return room[0];
}

template <typename T>
__global__ __launch_bounds__(256) void log_probs_kernel(LogProbs a) {
  __shared__ unsigned long long keys[256];
  __shared__ float numbers[256];
  __shared__ int counts[256];
  const int r = blockIdx.x;
  const T* row = reinterpret_cast<const T*>(a.logits) + (size_t)r * a.ld;
  float m = -INFINITY;
  for (int v = threadIdx.x; v < a.vocab; v += 256) m = fmaxf(m, logit(row + v));
  m = over_group(m, numbers, [](float x, float y) { return fmaxf(x, y); });
  const bool nothing = m == -INFINITY;
  const long long target = a.targets ? a.targets[r] : -1;
  const bool asked = target >= 0 && target < a.vocab;
  const float mine = asked ? logit(row + target) : 0.f;
  const unsigned long long my_key = asked ? key_of(mine, (int)target) : ~0ull;
  float s = 0.f, u = 0.f;
  int ahead = 0;
  for (int v = threadIdx.x; v < a.vocab; v += 256) {
    const float x = logit(row + v), d = x - (nothing ? 0.f : m), p = exp2_hw(d * kLog2e);
    s += p;
    u += p != 0.f ? p * d : 0.f;
    ahead += key_of(x, v) > my_key;
  }
  const auto add = [](auto x, auto y) { return x + y; };
  s = over_group(s, numbers, add);
  u = over_group(u, numbers, add);
  ahead = over_group(ahead, counts, add);
  const bool empty = nothing && s == 0.f;
  const float log_s = logf(s);
  if (threadIdx.x == 0) {
    if (a.entropy) a.entropy[r] = empty ? 0.f : log_s - u / s;
    if (a.targets) {
      a.log_probs[r] = !asked ? 0.f : empty ? -INFINITY : (mine - m) - log_s;
      a.ranks[r] = asked ? ahead : -1;
    }
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    unsigned long long best = 0;
    for (int v = threadIdx.x; v < a.vocab; v += 256) {
      const unsigned long long key = key_of(logit(row + v), v);
      if (key < last && key > best) best = key;
    }
    last = over_group(best, keys, [](unsigned long long x, unsigned long long y) { return x > y ? x : y; });
    if (threadIdx.x == 0) {
      const int id = (int)~(uint32_t)last;
      a.top_ids[(size_t)r * a.top + k] = id;
      a.top_log_probs[(size_t)r * a.top + k] = empty ? -INFINITY : (logit(row + id) - m) - log_s;
    }
  }
}

}  // namespace ajq
