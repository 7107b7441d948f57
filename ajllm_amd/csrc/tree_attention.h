// Attention of a tree of drafted tokens over a cache: each sees the committed rows and, of the tokens' own behind them, those whose bits its mask has.
//
//   out[b, t, h] = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c q . k_j - m),  c = log2(e) / sqrt(HD)
//
// All of a sequence's tokens see nearly the same rows, so that a key head's rows meet tokens * share queries as a matrix product's, by the ways of
// shared_attention.h: meet_few by tiles of 16 or 32 queries, meet_many by 64 or 128.  There the rows are one run; a block of 32 of them is seen by everybody, or (two
// or three at the end) by those queries whose bits say so: one shift of two mask words a query.
//
// Where tiles are few the rows are cut into parts, which a second launch puts together.  Sequences are of different lengths, and a launch of one round takes as long as
// its longest part: a number of runs, fixed by the host, is dealt out to the sequences by their lengths, which only the device knows (every workgroup
// works out the same).
#pragma once
#include "shared_attention.h"

namespace ajq {

struct TreeAttention : SharedAttention {   // (the prefix's caches are the sequences' own; prefix_blocks, prefix_parts 0)
  const uint32_t* masks;
  long long mask_batch, mask_token;
  int2* dealt;   // [batch] a sequence's first run, and how many it has
  int runs;      // parts of rows a key head (0: every sequence's rows are one)
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

// ---- dealing.  With n_b blocks of rows a sequence, R runs and B sequences, parts of Q blocks are too many if sum ceil(n_b / Q) > R; Q = sum n_b / (R - B) is always
// enough, sum n_b / R the least that can be.  Each lane tries a Q between the two, and the smallest that fits is taken.
constexpr int kMostDealt = 64;   // sequences: a lane each
struct Dealt {
  int sequence, part, parts, before, rows, there;   // (rows: 0 where no token is there)
};
__device__ __forceinline__ int parts_by(int blocks, float by) { return max(1, (int)ceilf((float)blocks * by - 1e-3f)); }
template <int kBlock>
__device__ __forceinline__ bool deal(const TreeAttention& a, int run, bool tells, Dealt& d) {
  if (a.batch == 1) {   // (every run is its)
    const long long at = read_uniform(a.rows) + (a.offset ? read_uniform(a.offset) : 0ll);
    d.there = a.counts ? held(read_uniform(a.counts), a.tokens) : a.tokens;
    d.sequence = 0;
    d.part = run;
    d.parts = a.runs;
    d.before = held_place(at);
    d.rows = d.there > 0 ? held(at + d.there, a.max_len) : 0;
    return true;
  }
  const int lane = threadIdx.x & 63, mine = min(lane, a.batch - 1);
  const long long first_row = a.rows[mine] + (a.offset ? *a.offset : 0ll);
  const int there = a.counts ? held(a.counts[mine], a.tokens) : a.tokens, before = held_place(first_row);
  const int rows = there > 0 ? held(first_row + there, a.max_len) : 0, blocks = lane < a.batch ? (rows + kBlock - 1) / kBlock : 0;
  const float total = wave_sum((float)blocks), least = total / (float)a.runs, enough = total * 1.0001f / (float)(a.runs - a.batch) + 1.f;
  float by = 1.f / fmaxf(1.f, ceilf(least + (enough - least) * (float)lane * (1.f / 63.f)));
  int sum = 0;
  for (int b = 0; b < a.batch; ++b) sum += parts_by(__builtin_amdgcn_readlane(blocks, b), by);
  const unsigned long long fits = __builtin_amdgcn_ballot_w64(sum <= a.runs);
  by = __uint_as_float((uint32_t)__builtin_amdgcn_readlane(__float_as_int(by), fits ? __builtin_ctzll(fits) : 63));
  const int parts = min(parts_by(blocks, by), 64);   // (a lane each in the merge)
  int b = 0, first = 0;
  for (; b < a.batch; ++b) {
    d.parts = __builtin_amdgcn_readlane(parts, b);
    if (run < first + d.parts) break;
    first += d.parts;
  }
  if (b == a.batch) return false;
  b = __builtin_amdgcn_readfirstlane(b);   // (all the same in every lane; said once more, since addresses have to be)
  d.sequence = b;
  d.part = __builtin_amdgcn_readfirstlane(run - first);
  d.parts = __builtin_amdgcn_readfirstlane(d.parts);
  d.before = __builtin_amdgcn_readlane(before, b);
  d.rows = __builtin_amdgcn_readlane(rows, b);
  d.there = __builtin_amdgcn_readlane(there, b);
  if (tells && d.part == 0 && threadIdx.x == 0) a.dealt[b] = int2{first, d.parts};
  return true;
}
// partial results: [runs, key heads, a sequence's queries of a key head]
__device__ __forceinline__ long long part_place(const TreeAttention& a, int run, int key_head, int n) {
  return ((long long)run * a.kv_heads + key_head) * (int)a.by_each.d + n;
}
template <typename CacheT>
__device__ __forceinline__ long long part_place(const TreeAttention& a, const Meeting<CacheT>& w, long long, int n) { return part_place(a, w.part, w.key_head, n); }
__device__ __forceinline__ long long part_place(const TreeAttention& a, const Walk<uint16_t>& w, long long, int n, int run) { return part_place(a, run, w.key_head, n); }

// a workgroup's run, key head and tile of queries; tiles that share rows are next to each other on one XCD
__device__ __forceinline__ bool find_turn(const TreeAttention& a, int& run, int& key_head, int& tile) {
  const int id = (int)blockIdx.x, at = (id & 7) + 8 * divide(id >> 3, a.by_own_tiles, tile);
  run = divide(at, a.by_kv_heads, key_head);
  return run < a.runs;
}
template <typename CacheT>
__device__ __forceinline__ void find_rows(const TreeAttention& a, Meeting<CacheT>& w) {
  if (a.runs == 0) find_rows(static_cast<const SharedAttention&>(a), w);
}

// A tile's queries and a part of the rows to a workgroup of WV waves (kWhole: all rows, and what comes out is the result).
template <int HD, typename QT, typename CacheT, int RT, int WV, bool kWhole>
__global__ __launch_bounds__(64 * WV, sizeof(CacheT) == 4 && RT == 2 && WV == 4 ? 1 : 2) void tree_attention_few_kernel(TreeAttention a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char shared_lds[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(pf_lds_char_t*)shared_lds;
  Meeting<CacheT> w;
  if constexpr (kWhole) {
    if (!find_meeting<CacheT, HD>(a, 16, 16 * RT, w)) return;
  } else {
    int tile;
    Dealt d;
    if (!find_turn(a, w.part, w.key_head, tile) || !deal<32>(a, w.part, w.key_head == 0 && tile == 0, d)) return;
    w.own = true;
    w.alone = false;
    w.outer = w.first_sequence = d.sequence;
    w.queries = (int)a.by_each.d;
    w.first = 16 * RT * tile;
    if (w.first >= d.there * (int)a.by_share.d) return;
    const size_t at = (size_t)d.sequence * a.cache_batch + (size_t)w.key_head * a.cache_head;
    w.keys = reinterpret_cast<const CacheT*>(a.keys) + at;
    w.values = reinterpret_cast<const CacheT*>(a.values) + at;
    w.before = d.before;
    const int per = ((d.rows + d.parts - 1) / d.parts + 31) & ~31;
    w.begin = (int)min((long long)d.rows, (long long)d.part * per);
    w.end = min(d.rows, w.begin + per);
  }
  meet_some<HD, QT, CacheT, RT, false, kWhole, WV>(a, w, shared_lds, lds0);
}
template <int HD, typename QT, int U, int WV>
__global__ __launch_bounds__(64 * WV, 2) void tree_attention_walk_kernel(TreeAttention a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char shared_lds[];
  WalkTurn turn;
  if (a.runs == 0) {
    const int id = (int)blockIdx.x, at = (id & 7) + 8 * divide(id >> 3, a.by_own_tiles, turn.tile);
    turn.sequence = divide(at, a.by_kv_heads, turn.key_head);
    if (turn.sequence >= a.batch) return;
    turn.part = turn.left_at = 0;
    turn.parts = 1;
  } else {
    Dealt d;
    if (!find_turn(a, turn.left_at, turn.key_head, turn.tile) || !deal<64>(a, turn.left_at, turn.key_head == 0 && turn.tile == 0, d)) return;
    if (16 * WV * U * turn.tile >= d.there * (int)a.by_share.d) return;
    turn.sequence = d.sequence;
    turn.part = d.part;
    turn.parts = d.parts;
  }
  walk_own<HD, QT, U, WV>(a, turn, a.runs > 0, (uint32_t)(uintptr_t)(pf_lds_char_t*)shared_lds);
}
template <int HD>
__global__ __launch_bounds__(256) void tree_attention_merge_kernel(TreeAttention a) {
  const long long place = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (place >= a.queries) return;
  int t, h, in_group;
  const int b = divide(divide((int)place, a.by_tokens, t), a.by_heads, h), key_head = divide(h, a.by_share, in_group);
  uint16_t* out = a.out + (((size_t)b * a.tokens + t) * a.heads + h) * HD;
  if (a.counts != nullptr && t >= a.counts[b]) {
    constexpr int kEach = HD == 128 ? 2 : 1;
    const int lane = threadIdx.x & 63;
    if (kEach * lane < HD) {
      if constexpr (kEach == 2) *reinterpret_cast<uint32_t*>(out + 2 * lane) = 0u;
      else out[lane] = 0;
    }
    return;
  }
  const int2 dealt = a.batch == 1 ? int2{0, a.runs} : a.dealt[b];
  const long long at = part_place(a, dealt.x, key_head, t * (int)a.by_share.d + in_group);
  put_together<HD>(a.part_ml + at, a.part_sums + at * HD, (size_t)a.kv_heads * (int)a.by_each.d, dealt.y, [&](bool& there, uint16_t*& to) __attribute__((always_inline)) {
    there = true;
    to = out;
  });
}

}  // namespace ajq
