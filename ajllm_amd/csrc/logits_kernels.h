// Logits ahead of the choice of a token: penalties for tokens that a row holds already, biases, masks of allowed tokens.
//
// A workgroup takes a slice of one row's vocabulary.  It keeps a word per token of the slice in LDS,
//   bits 0 .. 19  how often the token is among the row's tokens,   bit 20  whether it is in the prompt,   bits 21 .. 31  its bias slot + 1,
// fills them from the row's lists (whole numbers: no result depends on the order of the atomics), then walks the slice once.
#pragma once
#include "ajq_common.h"

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
  int slice;
};

__device__ __forceinline__ float logit_of(const float* p) { return *p; }
__device__ __forceinline__ float logit_of(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }

// Grid (rows, slices); `words` are a.slice words of LDS (none where the row has neither lists nor biases: kWords false).
template <typename T, bool kWords>
__global__ __launch_bounds__(1024) void adjust_logits_kernel(AdjustLogits a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t words[];
  __shared__ float sums[kWords ? kMaxBiases : 1];
  __shared__ int bias_at[kWords ? kMaxBiases : 1];
  const int b = blockIdx.x, t = threadIdx.x, threads = blockDim.x;
  const int base = blockIdx.y * a.slice, count = min(a.slice, a.vocab - base);
  if (kWords) {
    for (int i = t; i < count; i += threads) words[i] = 0u;
    __syncthreads();
    auto held = [&](const long long* counts, int stride, int most) {
      return counts ? (int)min(max(counts[(size_t)b * stride], 0ll), (long long)most) : most;
    };
    if (a.tokens) {
      const int n = held(a.token_counts, a.token_count_stride, a.max_tokens);
      for (int i = t; i < n; i += threads) {
        const long long at = a.tokens[(size_t)b * a.tokens_ld + i] - base;
        if (at >= 0 && at < count) atomicAdd(&words[at], 1u);
      }
    }
    if (a.prompt) {
      const int n = held(a.prompt_counts, a.prompt_count_stride, a.max_prompt);
      for (int i = t; i < n; i += threads) {
        const long long at = a.prompt[(size_t)b * a.prompt_ld + i] - base;
        if (at >= 0 && at < count) atomicOr(&words[at], kInPrompt);
      }
    }
    for (int i = t; i < a.biases; i += threads) {
      const long long at = a.bias_ids[(size_t)b * a.bias_ld + i] - base;
      bias_at[i] = at >= 0 && at < count ? (int)at : -1;
      sums[i] = a.bias[(size_t)b * a.bias_ld + i];
    }
    __syncthreads();
    // the first of a token's entries takes the sum of all of them, in their order
    float mine = 0.f;
    bool first = false;
    if (t < a.biases && bias_at[t] >= 0) {
      first = true;
      for (int j = 0; j < a.biases; ++j) {
        if (bias_at[j] != bias_at[t]) continue;
        if (j < t) first = false;
        mine += sums[j];
      }
    }
    __syncthreads();
    if (first) {
      sums[t] = mine;
      atomicOr(&words[bias_at[t]], (uint32_t)(t + 1) << 21);
    }
    __syncthreads();
  }
  const float repeat = a.repetition ? a.repetition[b] : 1.f, frequency = a.frequency ? a.frequency[b] : 0.f,
              presence = a.presence ? a.presence[b] : 0.f;
  const uint32_t* mask = nullptr;
  if (a.allowed) {
    const long long which = a.allowed_rows ? a.allowed_rows[b] : (long long)b;
    if (which >= 0 && which < a.masks) mask = a.allowed + which * a.allowed_ld;
  }
  const T* row = reinterpret_cast<const T*>(a.logits) + (size_t)b * a.ld + base;
  float* to = a.out + (size_t)b * a.out_ld + base;
  for (int i = t; i < count; i += threads) {
    float x = logit_of(row + i);
    if (kWords) {
      const uint32_t w = words[i];
      if (w) {
        const uint32_t n = w & (kInPrompt - 1);
        if (w & (kInPrompt | (kInPrompt - 1))) x = x > 0.f ? x / repeat : x * repeat;
        if (n) x -= frequency * (float)n + presence;
        if (w >> 21) x += sums[(w >> 21) - 1];
      }
    }
    if (mask && !((mask[(base + i) >> 5] >> ((base + i) & 31)) & 1u)) x = -INFINITY;
    to[i] = x;
  }
}

}  // namespace ajq
