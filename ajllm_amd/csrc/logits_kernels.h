// Logits ahead of the choice of a token: penalties for tokens that a row holds already, biases, masks of allowed tokens.
//
// A workgroup takes a slice of one row's vocabulary.  It asks for its logits, then keeps a word per token of the slice in LDS,
//   bits 0 .. 19  how often the token is among the row's tokens,   bit 20  whether it is in the prompt,   bits 21 .. 31  its bias slot + 1,
// fills them from the row's lists (whole numbers: no result depends on the order of the atomics) while the logits are on their way, and
// puts both together, four tokens a lane at a time.  What bounds it is memory: a row is read and written once; its lists are read by
// every slice, from L2 (slices of a row run next to each other on one XCD).  256 rows of 128256 fp32 logits with 9216 listed tokens and a mask each (281 MB)
// 65.6 us = 4.3 TB/s, 32 rows with 2560 11.4 us, one of 32000 4.2: a launch and two round trips, the lists' and the logits'.  In place only what changes is read, but behind the lists:
// whole calls, 256 rows 51 us (60 elsewhere) without masks, 72 (66) with masks that leave half of the tokens; 32 rows 10.1 (10.5) and 13.1 (11.4).
#pragma once
#include "lane_rows.h"

namespace ajq {

constexpr int kMaxBiases = 1024, kMaxHistory = (1 << 20) - 1;
constexpr uint32_t kInPrompt = 1u << 20;

struct AdjustLogits {
  const void* logits;
  float* out;
  const long long *tokens, *token_counts, *prompt, *prompt_counts;
  const float *repetition, *frequency, *presence;
  const long long* bias_ids;
  const float* bias;
  const uint32_t* allowed;
  const long long* allowed_rows;
  long long ld, out_ld, tokens_ld, prompt_ld, bias_ld, allowed_ld;
  int vocab, max_tokens, max_prompt, biases, masks, token_count_stride, prompt_count_stride;
  int batch, slice, slices;
};

constexpr int kSliceThreads = 1024, kSlicePieces = 4;   // lanes, and pieces of four tokens a lane: slices of up to 16384 tokens

// Four logits by one load, wherever they lie (rows of an odd vocabulary begin anywhere; the hardware takes any address); fewer at a row's end.
// A row goes past L2, which the lists are read from.
typedef float f32x4u_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2u_t __attribute__((ext_vector_type(2), aligned(2)));
__device__ __forceinline__ f32x4_t load_logits(const float* p, int there) {
  if (there >= 4) return __builtin_nontemporal_load(reinterpret_cast<const f32x4u_t*>(p));
  return f32x4_t{p[0], there > 1 ? p[1] : 0.f, there > 2 ? p[2] : 0.f, 0.f};
}
__device__ __forceinline__ f32x4_t load_logits(const uint16_t* p, int there) {
  u32x2_t v;
  if (there >= 4) v = __builtin_nontemporal_load(reinterpret_cast<const u32x2u_t*>(p));
  else v = u32x2_t{p[0] | (there > 1 ? (uint32_t)p[1] << 16 : 0u), there > 2 ? p[2] : 0u};
  return f32x4_t{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xFFFF0000u)};
}
__device__ __forceinline__ void store_logits(float* p, int there, f32x4_t x) {
  if (there >= 4) {
    __builtin_nontemporal_store(x, reinterpret_cast<f32x4u_t*>(p));
  } else {
    p[0] = x[0];
    if (there > 1) p[1] = x[1];
    if (there > 2) p[2] = x[2];
  }
}
// fn(id) for the first n of a list of `most`.  The first ids are asked for before n is known (ask), four a lane.
struct Ids {
  static constexpr int kAtOnce = 4;
  long long id[kAtOnce];
};
__device__ __forceinline__ void ask_ids(const long long* ids, int first, int most, Ids& got) {
#pragma unroll
  for (int i = 0; i < Ids::kAtOnce; ++i) got.id[i] = ids[min(first + i * (int)blockDim.x, most - 1)];
}
template <typename F>
__device__ __forceinline__ void each_id(const long long* ids, int n, Ids& got, F&& fn) {
  for (int first = threadIdx.x;;) {
#pragma unroll
    for (int i = 0; i < Ids::kAtOnce; ++i)
      if (first + i * (int)blockDim.x < n) fn(got.id[i]);
    first += Ids::kAtOnce * (int)blockDim.x;
    if (first >= n) break;
    ask_ids(ids, first, n, got);
  }
}

// kWords: rows have lists or biases (a.slice words of LDS); kInPlace: logits are the results, and only what changes is read and written.
template <typename T, bool kWords, bool kInPlace>
__global__ __launch_bounds__(kSliceThreads, 8) void adjust_logits_kernel(AdjustLogits a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t words[];
  __shared__ float sums[kWords ? kMaxBiases : 1];
  __shared__ int bias_at[kWords ? kMaxBiases : 1];
  __shared__ int again;   // whether a token is biased twice
  const int t = threadIdx.x, threads = blockDim.x;
  const int turn = (int)(blockIdx.x >> 3) / a.slices;
  const int b = 8 * turn + (int)(blockIdx.x & 7), base = ((int)(blockIdx.x >> 3) - turn * a.slices) * a.slice;
  if (b >= a.batch) return;
  const int count = min(a.slice, a.vocab - base);
  const T* row = reinterpret_cast<const T*>(a.logits) + (size_t)b * a.ld + base;
  f32x4_t x[kSlicePieces] = {};
  if (!kInPlace) {
#pragma unroll
    for (int i = 0; i < kSlicePieces; ++i) {
      const int at = 4 * (t + i * threads);
      x[i] = at < count ? load_logits(row + at, count - at) : f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  }
  const long long *tokens = nullptr, *prompt = nullptr, *bias_ids = nullptr;
  const float* bias = nullptr;
  Ids mine, given;
  long long bias_id = -1;
  float bias_by = 0.f;
  if (kWords) {
    if (a.tokens) ask_ids(tokens = a.tokens + (size_t)b * a.tokens_ld, t, a.max_tokens, mine);
    if (a.prompt) ask_ids(prompt = a.prompt + (size_t)b * a.prompt_ld, t, a.max_prompt, given);
    if (a.biases) {
      bias_ids = a.bias_ids + (size_t)b * a.bias_ld;
      bias = a.bias + (size_t)b * a.bias_ld;
      bias_id = bias_ids[min(t, a.biases - 1)];
      bias_by = bias[min(t, a.biases - 1)];
    }
  }
  const uint32_t* mask = nullptr;
  if (a.allowed) {
    const long long which = a.allowed_rows ? a.allowed_rows[b] : (long long)b;
    if (which >= 0 && which < a.masks) mask = a.allowed + which * a.allowed_ld;
  }
  uint32_t allowed[kSlicePieces];
#pragma unroll
  for (int i = 0; i < kSlicePieces; ++i) {
    const int at = 4 * (t + i * threads);
    allowed[i] = mask && at < count ? mask[(base + at) >> 5] >> (at & 31) : 15u;   // (slices begin on boundaries of 32)
  }
  const float repeat = a.repetition ? a.repetition[b] : 1.f, frequency = a.frequency ? a.frequency[b] : 0.f,
              presence = a.presence ? a.presence[b] : 0.f;
  if (kWords) {
    for (int i = 4 * t; i < a.slice; i += 4 * threads) *reinterpret_cast<u32x4_t*>(words + i) = u32x4_t{0u, 0u, 0u, 0u};
    if (t == 0) again = 0;
    __syncthreads();
    auto held = [&](const long long* counts, int stride, int most) {
      return counts ? (int)min(max(counts[(size_t)b * stride], 0ll), (long long)most) : most;
    };
    if (tokens)
      each_id(tokens, held(a.token_counts, a.token_count_stride, a.max_tokens), mine, [&](long long id) {
        const long long at = id - base;
        if (at >= 0 && at < count) atomicAdd(&words[at], 1u);
      });
    if (prompt)
      each_id(prompt, held(a.prompt_counts, a.prompt_count_stride, a.max_prompt), given, [&](long long id) {
        const long long at = id - base;
        if (at >= 0 && at < count) atomicOr(&words[at], kInPrompt);
      });
    __syncthreads();
    if (a.biases) {
      // a token's slot is that of its first entry, which takes the sum of all of them, in their order.  (Slot kMaxBiases - i for entry i: the largest is the
      // first.  The low bits are settled by now.)
      for (int i = t; i < a.biases; i += threads) {
        const long long at = (i == t ? bias_id : bias_ids[i]) - base;
        const bool here = at >= 0 && at < count;
        bias_at[i] = here ? (int)at : -1;
        sums[i] = i == t ? bias_by : bias[i];
        if (here) atomicMax(&words[at], (words[at] & ((1u << 21) - 1)) | ((uint32_t)(kMaxBiases - i) << 21));
      }
      __syncthreads();
      for (int i = t; i < a.biases; i += threads)
        if (bias_at[i] >= 0 && words[bias_at[i]] >> 21 != (uint32_t)(kMaxBiases - i)) again = 1;
      __syncthreads();
      if (again) {
        for (int first = 0; first < a.biases; first += threads) {
          const int i = first + t;
          const bool take = i < a.biases && bias_at[i] >= 0 && words[bias_at[i]] >> 21 == (uint32_t)(kMaxBiases - i);
          float sum = 0.f;
          if (take) {
            for (int j = i; j < a.biases; ++j)
              if (bias_at[j] == bias_at[i]) sum += sums[j];
          }
          __syncthreads();
          if (take) sums[i] = sum;   // (no entry of a later round reads it)
          __syncthreads();
        }
      }
    }
  }
  float* to = a.out + (size_t)b * a.out_ld + base;
#pragma unroll
  for (int i = 0; i < kSlicePieces; ++i) {
    const int at = 4 * (t + i * threads);
    if (at < count) {
      u32x4_t w = u32x4_t{0u, 0u, 0u, 0u};
      if (kWords) w = *reinterpret_cast<const u32x4_t*>(words + at);
      const bool changed = (w.x | w.y | w.z | w.w) != 0u || (allowed[i] & 15u) != 15u;
      f32x4_t v = x[i];
      if (kInPlace && changed) v = load_logits(row + at, count - at);
      if (kWords) {
        // (few of a wave's tokens have a word: one after the other, a lane its next one)
        uint32_t todo = (w.x != 0u ? 1u : 0u) | (w.y != 0u ? 2u : 0u) | (w.z != 0u ? 4u : 0u) | (w.w != 0u ? 8u : 0u);
        while (todo) {
          const bool second = (todo & 1u) == 0u, upper = (todo & 3u) == 0u, last = (todo & 7u) == 0u;
          const uint32_t word = upper ? (last ? w.w : w.z) : (second ? w.y : w.x);
          float y = upper ? (last ? v.w : v.z) : (second ? v.y : v.x);
          const uint32_t n = word & (kInPrompt - 1);
          if (word & (kInPrompt | (kInPrompt - 1))) y = y > 0.f ? y / repeat : y * repeat;
          if (n) y -= frequency * (float)n + presence;
          if (word >> 21) y += sums[kMaxBiases - (word >> 21)];
          v.x = second ? v.x : y;
          v.y = second && !upper ? y : v.y;
          v.z = upper && !last ? y : v.z;
          v.w = last ? y : v.w;
          todo &= todo - 1;
        }
      }
      v.x = allowed[i] & 1u ? v.x : -INFINITY;
      v.y = allowed[i] & 2u ? v.y : -INFINITY;
      v.z = allowed[i] & 4u ? v.z : -INFINITY;
      v.w = allowed[i] & 8u ? v.w : -INFINITY;
      if (!kInPlace || changed) store_logits(to + at, count - at, v);
    }
  }
}

}  // namespace ajq
