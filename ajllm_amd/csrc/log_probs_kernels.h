// Log probabilities of given tokens, entropies, and the first tokens in the order of their logits.
//
//   log p_t = (x_t - m) - log s,   H = log s - u / s,   m = max x_v,   s = sum e^(x_v - m),   u = sum e^(x_v - m) (x_v - m)
//
// A workgroup takes a slice of one row, up to 128 KiB, into its registers at once, so that everything behind the maximum is worked out of them and memory
// is read once.  Slices' (m, s, u, tokens ahead) and first tokens are put together by a second launch where a row has several.
//
// The first `top` of a slice: lanes 128 apart are a group, and every group knows its largest logit and the 16 bytes that it first has it in.  The top-th of these 128 is
// a border that at least `top` tokens reach, and only the groups that lead it have others that do: some top * (1 + top / 256) of them in a row without order, 16 bytes'
// worth of tokens for each of `top` in one that is all alike or sorted.  Their pieces gather in LDS, a lane takes a token, each counts those ahead of itself, and
// that is its place.  Where they are more than LDS is set aside for (a row made to be so), `top` rounds over the slice find them instead.
#pragma once
#include "lane_rows.h"
#include <type_traits>

namespace ajq {

constexpr int kMostTop = 64, kLogPieces = 8, kGroups = 128, kHits = 512, kGathered = 1024;   // (at least the lanes of a workgroup)
struct LogProbs {
  const void* logits;
  const long long* targets;
  float *log_probs, *entropy, *top_log_probs;
  long long *ranks, *top_ids;
  f32x4_t* parts;               // [rows, slices] m, s, u, tokens ahead of the target (a whole number's bits)
  float* mine;                  // [rows] the target's logit
  unsigned long long* firsts;   // [rows, slices, top]
  long long ld;
  int rows, vocab, top, slice, slices;
};

// The order of the tokens as whole numbers: larger logits first (NaN ahead of all, -0 as 0), then smaller ids.  0 is no token's.
__device__ __forceinline__ unsigned long long key_of(float x, int id) {
  const uint32_t bits = __float_as_uint(x + 0.f);
  const uint32_t order = x != x ? 0xFFFFFFFFu : bits ^ ((uint32_t)((int)bits >> 31) | 0x80000000u);
  return (unsigned long long)order << 32 | (uint32_t)~id;
}
__device__ __forceinline__ int id_of(unsigned long long key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float logit_of(unsigned long long key) {
  const uint32_t order = (uint32_t)(key >> 32);
  return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}
__device__ __forceinline__ unsigned long long larger(unsigned long long x, unsigned long long y) { return x > y ? x : y; }

__device__ __forceinline__ float logit(const float* p) { return *p; }
__device__ __forceinline__ float logit(const uint16_t* p) { return __uint_as_float((uint32_t)*p << 16); }
template <typename T> constexpr int kPiece = 16 / (int)sizeof(T);   // logits of 16 bytes
template <typename T>
__device__ __forceinline__ float logit(const u32x4_t& raw, int e) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(raw[e]);
  return __uint_as_float(e & 1 ? raw[e >> 1] & 0xFFFF0000u : raw[e >> 1] << 16);
}
// the logits of a piece from `first` to `last`, -inf for the others
template <typename T>
__device__ __forceinline__ u32x4_t load_some(const T* p, int first, int last) {
  uint32_t w[kPiece<T>];
#pragma unroll
  for (int e = 0; e < kPiece<T>; ++e) w[e] = e >= first && e <= last ? reinterpret_cast<const std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>*>(p)[e] : sizeof(T) == 4 ? 0xFF800000u : 0xFF80u;
  if constexpr (sizeof(T) == 4) return u32x4_t{w[0], w[1], w[2], w[3]};
  else return u32x4_t{w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16};
}

__device__ __forceinline__ float wave_most(float v) {
  v = quad_max(v);   // over lanes l, l ^ 16, l ^ 32, l ^ 48
  v = fmaxf(v, row_ror<8>(v));
  v = fmaxf(v, row_ror<4>(v));
  v = fmaxf(v, row_ror<2>(v));
  return fmaxf(v, row_ror<1>(v));
}

// numbers that all lanes have, kept where such numbers are (the logits leave no registers for them)
__device__ __forceinline__ float uniform(float v) { return __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane(__float_as_int(v))); }
__device__ __forceinline__ unsigned long long uniform(unsigned long long v) {
  return (unsigned long long)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v) | (unsigned long long)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32)) << 32;
}

// What is known of a row, or of a slice of it.
struct RowSums {
  float m, s, u;   // (m: 0 where everything is -inf)
  int ahead;
  bool nothing;
};
__device__ __forceinline__ float log_prob(float x, const RowSums& r, float log_s) { return r.nothing ? -INFINITY : (x - r.m) - log_s; }
__device__ __forceinline__ void leave_row(const LogProbs& a, int row, const RowSums& r, float log_s, bool asked, float mine) {
  a.entropy[row] = r.nothing ? 0.f : log_s - r.u / r.s;
  if (a.targets) {
    a.log_probs[row] = asked ? log_prob(mine, r, log_s) : 0.f;
    a.ranks[row] = asked ? min(r.ahead, a.vocab - 1) : -1;
  }
}

template <typename T, int LANES, bool kRank, bool kTop>
__global__ __launch_bounds__(LANES, 8) void log_probs_kernel(LogProbs a) {
  constexpr int E = kPiece<T>, W = LANES / 64, kRound = LANES * E;
  __shared__ __attribute__((aligned(16))) float most[W], sums[W], spreads[W];
  __shared__ int aheads[W], hits, gathered, places[kTop ? kGroups : 1], hit_places[kTop ? kHits : 1];
  __shared__ __attribute__((aligned(16))) u32x4_t hit_pieces[kTop ? kHits : 1];
  __shared__ __attribute__((aligned(16))) unsigned long long groups[kTop ? kGroups : 1], found[kTop ? kGathered : 1];   // (found: at first the lanes' own)
  const int t = threadIdx.x, wave = t >> 6;
  const int r = (int)blockIdx.x / a.slices, part = (int)blockIdx.x - r * a.slices, base = part * a.slice;
  const T* row = reinterpret_cast<const T*>(a.logits) + (size_t)r * a.ld;
  const T* slice = row + base;
  const int count = min(a.slice, a.vocab - base);
  // Places go by 16 bytes, wherever the slice begins (a row of an odd vocabulary begins anywhere; pieces across such borders take a quarter longer): token base + n is in
  // place shift + n.
  const int shift = (int)((reinterpret_cast<uintptr_t>(slice) & 15u) / sizeof(T)), places_end = shift + count;
  slice -= shift;
  constexpr uint32_t kNone = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
  u32x4_t x[kLogPieces];
#pragma unroll
  for (int i = 0; i < kLogPieces; ++i) {
    const int at = t * E + i * kRound;
    x[i] = u32x4_t{kNone, kNone, kNone, kNone};
    if (at >= shift && at + E <= places_end) x[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(slice + at));
  }
  // the piece that the slice begins in, and that it ends in
  if (t == 0 && shift > 0) x[0] = load_some(slice, shift, places_end - 1);
  const int last = (places_end - 1) / E;
  if (places_end % E != 0 && t == last % LANES && last * E >= shift) {
    const u32x4_t v = load_some(slice + last * E, 0, (places_end - 1) % E);
#pragma unroll
    for (int i = 0; i < kLogPieces; ++i)
      if (i == last / LANES) x[i] = v;
  }
  bool asked = false;
  float mine = 0.f;
  int ahead = 0, target = 0;   // (ahead: the wave's; votes, since a sum a lane is one vector instruction a token more: 45 us instead of 39 for 1030 x 64086 bf16)
  if constexpr (kRank) {
    const long long given = a.targets[r];
    asked = given >= 0 && given < a.vocab;
    const long long off = given - base;
    const bool here = off >= 0 && off < count;
    // its place, or one in front of all the slice's pieces or behind them
    target = here ? shift + (int)off : off < 0 ? 0 : (last + 1) * E;
    if (asked) mine = uniform(logit(row + given));
    // of the target's own piece the tokens in front of it that have the same logit
    bool tied = false;
    if (asked && here && t < E - 1) {
      const int at = target / E * E + t;
      if (at >= shift && at < target) tied = logit(slice + at) == mine;
    }
    ahead = __builtin_popcountll(__builtin_amdgcn_ballot_w64(tied));
    // (what fills up the pieces that the slice begins and ends in counts below where they are in front of a target that is -inf itself)
    if (asked && t < 64 && mine == -INFINITY) ahead -= (target >= E ? shift : 0) + (target >= places_end ? (last + 1) * E - places_end : 0);
    ahead = __builtin_amdgcn_readfirstlane(ahead);
  }
  if constexpr (kTop) {
    if (t == 0) hits = gathered = 0;
    if (t < kGroups) places[t] = 0;
  }

  // ---- the maximum
  auto piece_top = [&](int i) __attribute__((always_inline)) {
    float v = logit<T>(x[i], 0);
#pragma unroll
    for (int e = 1; e < E; ++e) v = fmaxf(v, logit<T>(x[i], e));
    return v;
  };
  float top = -INFINITY;
  int first = 0;   // the piece of the lane's that first has its largest logit (none: NaN in its first, which is ahead of all)
#pragma unroll
  for (int i = 0; i < kLogPieces; ++i)
    if (i * kRound < places_end) {
      const float v = piece_top(i);
      if (kTop) first = v > top ? i : first;
      top = fmaxf(top, v);
    }
  const float lane_top = top;
  top = wave_most(top);
  if ((t & 63) == 0) most[wave] = top;
  if constexpr (kTop) {
    // of the lane's tokens one at least is not behind the last of that piece, and none is ahead of its first
    const int at = t * E + first * kRound;
    found[t] = at < places_end ? key_of(lane_top, base - shift + at + E - 1) : 0ull;
  }
  __syncthreads();
  if constexpr (kTop) {
    if (t < kGroups) {
      unsigned long long key = larger(found[t], kGroups - t);   // (of an empty group a number below every token's, its own)
#pragma unroll 2
      for (int i = kGroups; i < LANES; i += kGroups) key = larger(key, found[t + i]);
      groups[t] = key;
    }
    __syncthreads();
  }
  RowSums sum;
#pragma unroll
  for (int w = 0; w < W; ++w) top = fmaxf(top, most[w]);
  top = uniform(top);
  sum.m = top == -INFINITY ? 0.f : top;

  // ---- sums
  const float lower = asked ? mine : 0.f;
  const uint32_t bits = __float_as_uint(lower + 0.f);
  // the number just below the target's logit (of -inf none: no number is not above it)
  const float below = __uint_as_float(bits == 0u ? 0x80000001u : (int)bits > 0 ? bits - 1u : bits + 1u);
  float s = 0.f, u = 0.f;
  int end = places_end;
  asm volatile("" : "+s"(end));   // (here and below what has been worked out of the logits, or which of them there are, is not kept beside them but worked out again)
  const int ahead_of_target = target - (t * E + E - 1);
#pragma unroll
  for (int i = 0; i < kLogPieces; ++i)
    if (i * kRound < end) {
      asm volatile("" : "+v"(x[i]));
      const float than = i * kRound < ahead_of_target ? below : lower;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float v = logit<T>(x[i], e), d = v - sum.m, p = exp2_hw(d * kLog2e);
        s += p;
        u = __builtin_fmaf(p, fmaxf(d, -1e30f), u);   // (nothing of -inf)
        if constexpr (kRank) ahead += __builtin_popcountll(__builtin_amdgcn_ballot_w64(!(v <= than)));
      }
    }
  s = wave_sum(s);
  u = wave_sum(u);
  if ((t & 63) == 0) {
    sums[wave] = s;
    spreads[wave] = u;
    aheads[wave] = ahead;
  }
  // ---- a group's place among the others: a lane counts a share of them
  if constexpr (kTop) {
    constexpr int kShare = kGroups * kGroups / LANES;
    const unsigned long long key = groups[t % kGroups];
    int before = 0;
#pragma unroll 4   // (more would not leave the logits their registers)
    for (int i = 0; i < kShare; ++i) before += groups[t / kGroups * kShare + i] > key;
    atomicAdd(&places[t % kGroups], before);
  }
  __syncthreads();
  sum.s = sum.u = 0.f;
  sum.ahead = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    sum.s += sums[w];
    sum.u += spreads[w];
    sum.ahead += aheads[w];
  }
  sum.s = uniform(sum.s);
  sum.nothing = top == -INFINITY && sum.s == 0.f;
  const bool whole = a.slices == 1;
  const float log_s = uniform(logf(sum.s));
  if (t == 0) {
    if (whole) leave_row(a, r, sum, log_s, asked, mine);
    else a.parts[blockIdx.x] = f32x4_t{top, sum.s, sum.u, __int_as_float(sum.ahead)};
    if (kRank && !whole && part == 0) a.mine[r] = mine;
  }
  if constexpr (kTop) {
    // the border: the group in place top - 1
    const int lane = t & 63;
    const unsigned long long low = __builtin_amdgcn_ballot_w64(places[lane] == a.top - 1), high = __builtin_amdgcn_ballot_w64(places[64 + lane] == a.top - 1);
    const unsigned long long least = uniform(groups[low ? __builtin_ctzll(low) : 64 + __builtin_ctzll(high)]);
    const size_t to = (size_t)blockIdx.x * a.top;
    auto leave = [&](int place, unsigned long long key) {
      if (whole) {
        a.top_ids[to + place] = id_of(key);
        a.top_log_probs[to + place] = log_prob(logit_of(key), sum, log_s);
      } else {
        a.firsts[to + place] = key;
      }
    };
    // the lanes, and their pieces, that may hold such tokens: the largest logit with the first id reaches it
    int l = t, end = places_end;
    asm volatile("" : "+v"(l), "+s"(end));
    auto reaches = [&](float v, int at) { return at < end && key_of(v, base + max(at - shift, 0)) >= least; };
    if (reaches(lane_top, l * E + first * kRound)) {
#pragma unroll
      for (int i = 0; i < kLogPieces; ++i)
        if (i * kRound < end && reaches(piece_top(i), l * E + i * kRound)) {
          const int n = atomicAdd(&hits, 1);
          if (n < kHits) {
            hit_pieces[n] = x[i];
            hit_places[n] = l * E + i * kRound;
          }
        }
    }
    __syncthreads();
    const int some = hits;
    for (int n = t; n < min(some, kHits) * E; n += LANES) {
      const int id = hit_places[n / E] + n % E - shift;
      const unsigned long long key = key_of(logit(reinterpret_cast<const T*>(hit_pieces) + n), base + id);
      if (id >= 0 && id < count && key >= least) {
        const int to = atomicAdd(&gathered, 1);
        if (to < kGathered) found[to] = key;
      }
    }
    __syncthreads();
    const int many = gathered;
    if (some <= kHits && many <= kGathered) {
      for (int n = t; n < many; n += LANES) {
        const unsigned long long key = found[n];
        int place = 0;
#pragma unroll 8
        for (int i = 0; i < many; ++i) place += found[i] > key;
        if (place < a.top) leave(place, key);
      }
      if (!whole)   // (a slice that has fewer tokens than that)
        for (int n = many + t; n < a.top; n += LANES) a.firsts[to + n] = 0ull;
    } else {
      unsigned long long before = ~0ull;
#pragma unroll 1
      for (int k = 0; k < a.top; ++k) {
        unsigned long long best = 0ull;
#pragma unroll 1
        for (int id = t; id < count; id += LANES) {
          const unsigned long long key = key_of(logit(row + base + id), base + id);
          if (key < before) best = larger(best, key);
        }
        __syncthreads();
        found[t] = best;
        for (int n = LANES / 2; n > 0; n >>= 1) {
          __syncthreads();
          if (t < n) found[t] = larger(found[t], found[t + n]);
        }
        __syncthreads();
        before = found[0];
        if (t == 0) leave(k, before);
      }
    }
  }
}

// ---- a row's slices put together, a workgroup a row.  With S slices, the least of the tokens in place ceil(top / S) of theirs is a border that `top` tokens reach,
// and so is the first of those in place `top`; the tokens that reach both (twice as many or so; the second keeps out what a mask has left nothing of) gather, and each
// counts the ones ahead of itself.
constexpr int kMergeKeys = 2048;
__global__ __launch_bounds__(256) void log_probs_merge_kernel(LogProbs a) {
  __shared__ __attribute__((aligned(16))) unsigned long long keys[kMergeKeys];
  __shared__ int gathered;
  const int r = blockIdx.x, t = threadIdx.x, lane = t & 63;
  const f32x4_t* parts = a.parts + (size_t)r * a.slices;
  const unsigned long long* from = a.firsts + (size_t)r * a.slices * a.top;
  const int many = a.slices * a.top;
  if (t == 0) gathered = 0;
  const long long target = a.targets ? a.targets[r] : -1;
  const float mine = a.targets ? a.mine[r] : 0.f;
  // (every wave the same)
  float top = -INFINITY;
  unsigned long long least = ~0ull, first_of_last = 0ull;
  const int place_of_all = (a.top + a.slices - 1) / a.slices - 1;
  for (int n = lane; n < a.slices; n += 64) {
    top = fmaxf(top, parts[n][0]);
    if (a.top) {
      const unsigned long long key = from[n * a.top + place_of_all];
      least = key < least ? key : least;
      first_of_last = larger(first_of_last, from[n * a.top + a.top - 1]);
    }
  }
  top = wave_most(top);
  RowSums sum;
  sum.m = top == -INFINITY ? 0.f : top;
  sum.s = sum.u = 0.f;
  sum.ahead = 0;
  for (int n = lane; n < a.slices; n += 64) {
    const f32x4_t p = parts[n];
    const float d = p[0] - sum.m, w = exp2_hw(d * kLog2e);
    sum.s += p[1] * w;
    sum.u += w == 0.f ? 0.f : w * (p[2] + p[1] * d);
    sum.ahead += __float_as_int(p[3]);
  }
  sum.s = wave_sum(sum.s);
  sum.u = wave_sum(sum.u);
#pragma unroll
  for (int n = 32; n > 0; n >>= 1) sum.ahead += __shfl_xor(sum.ahead, n);
  sum.nothing = top == -INFINITY && sum.s == 0.f;
  const float log_s = logf(sum.s);
  if (t == 0) leave_row(a, r, sum, log_s, target >= 0 && target < a.vocab, mine);
  if (a.top == 0) return;
#pragma unroll
  for (int n = 32; n > 0; n >>= 1) {
    const unsigned long long other = __shfl_xor(least, n);
    least = other < least ? other : least;
    first_of_last = larger(first_of_last, __shfl_xor(first_of_last, n));
  }
  least = larger(least, first_of_last);
  auto leave = [&](int place, unsigned long long key) {
    if (place >= a.top) return;
    a.top_ids[(size_t)r * a.top + place] = id_of(key);
    a.top_log_probs[(size_t)r * a.top + place] = log_prob(logit_of(key), sum, log_s);
  };
  __syncthreads();
  for (int n = t; n < many; n += blockDim.x) {
    const unsigned long long key = from[n];
    if (key < least || key == 0ull) continue;
    const int to = atomicAdd(&gathered, 1);
    if (to < kMergeKeys) keys[to] = key;
  }
  __syncthreads();
  const int some = gathered;
  if (some <= kMergeKeys) {
    for (int n = t; n < some; n += blockDim.x) {
      const unsigned long long key = keys[n];
      int place = 0;
#pragma unroll 8
      for (int i = 0; i < some; ++i) place += keys[i] > key;
      leave(place, key);
    }
    return;
  }
  // (many slices with much the same tokens) a token's place in its slice and, of every other slice, how many are ahead of it
  for (int n = t; n < many; n += blockDim.x) {
    const unsigned long long key = from[n];
    if (key < least || key == 0ull) continue;
    const int own = n / a.top;
    int place = n - own * a.top;
    for (int other = 0; other < a.slices && place < a.top; ++other) {
      if (other == own) continue;
      int low = 0, high = a.top;   // the first of its places that is not ahead
      while (low < high) {
        const int middle = (low + high) >> 1;
        if (from[other * a.top + middle] > key) low = middle + 1;
        else high = middle;
      }
      place += low;
    }
    leave(place, key);
  }
}

}  // namespace ajq
