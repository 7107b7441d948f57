// Attention of a tree of drafted tokens over a cache: each sees the committed rows and, of the tokens' own behind them, those whose bits its mask has.
//
//   out[b, t, h] = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c q . k_j - m),  c = log2(e) / sqrt(HD)
//
// All of a sequence's tokens see nearly the same rows, so that a key head's rows meet tokens * share queries as a matrix product's, by the ways of
// shared_attention.h: meet_few by tiles of 16 or 32 queries, meet_many by 64, 128 or 256; many queries on fp32 rows have a way of their own here.  The rows are one
// run; a block of 32 of them is seen by everybody, or (two or three at the end) by those queries whose bits say so: one shift of two mask words a query.
//
// Where tiles are few the rows are cut into parts, which a second launch puts together.  Sequences are of different lengths, and a launch of one round takes as long as
// its longest part: a number of runs, fixed by the host, is dealt out to the sequences by their lengths, which only the device knows (every workgroup
// works out the same).
#pragma once
#include "shared_attention.h"
#include "tree_plan.h"   // kMostDealt

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

// A workgroup's tile of queries and its part of the rows (kWhole: all of them, and what comes out is the result).  False: none, and nothing to leave.
template <typename CacheT, int HD, bool kWhole>
__device__ __forceinline__ bool find_tile(const TreeAttention& a, int queries, Meeting<CacheT>& w) {
  if constexpr (kWhole) return find_meeting<CacheT, HD>(a, 16, queries, w);
  int tile;
  Dealt d;
  if (!find_turn(a, w.part, w.key_head, tile) || !deal<32>(a, w.part, w.key_head == 0 && tile == 0, d)) return false;
  w.own = true;
  w.alone = false;
  w.outer = w.first_sequence = d.sequence;
  w.queries = (int)a.by_each.d;
  w.first = queries * tile;
  if (w.first >= d.there * (int)a.by_share.d) return false;
  const size_t at = (size_t)d.sequence * a.cache_batch + (size_t)w.key_head * a.cache_head;
  w.keys = reinterpret_cast<const CacheT*>(a.keys) + at;
  w.values = reinterpret_cast<const CacheT*>(a.values) + at;
  w.before = d.before;
  const int per = ((d.rows + d.parts - 1) / d.parts + 31) & ~31;
  w.begin = (int)min((long long)d.rows, (long long)d.part * per);
  w.end = min(d.rows, w.begin + per);
  return true;
}

template <int HD, typename QT, typename CacheT, int RT, int WV, bool kWhole>
__global__ __launch_bounds__(64 * WV, sizeof(CacheT) == 4 && RT == 2 && WV == 4 ? 1 : 2) void tree_attention_few_kernel(TreeAttention a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char shared_lds[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(pf_lds_char_t*)shared_lds;
  Meeting<CacheT> w;
  if (!find_tile<CacheT, HD, kWhole>(a, 16 * RT, w)) return;
  meet_some<HD, QT, CacheT, RT, false, kWhole, WV>(a, w, shared_lds, lds0);
}

// ---- Many queries on fp32 rows: 16 RT to each of four waves, all on the same blocks of 32 rows.  What bounds meet_few there is that every wave splits its rows
// into two bf16 halves for its own queries; here the workgroup does so once: a block's pieces go from memory to the lanes' registers, and from there, as halves, to one of two
// stages of LDS (one barrier a block), while the next block's are on their way.  Products as there: scores of three (bf16 queries: two), results of two.
// Fp32 queries, us (by meet_few's best form; sequences have from half of these tokens and rows on): 7 x 69 of 32 heads of 128 behind up to 112 rows 18 (38); 7 x 100 behind 1000 64 (119); 8 x 64 of 32 / 8 behind 8000 159 (372), in 64
// parts; 12 x 25 of 12 heads of 64 behind 1500 22.6 (22.8).  350 calls with more than 16 queries a key head: 24 % less than without it if the faster is taken, 19 % as chosen.
// Bound by a wave's own work still: 80 MFMAs of 16 cycles, 64 pieces of 16 bytes from LDS and some 400 vector instructions a block, nothing of one block beside another's.
template <int HD> constexpr int laid_lds_bytes() { return 2 * 4 * 32 * 2 * HD; }   // stages; keys and values, each in halves
template <int HD, typename QT, int RT, bool kWhole>
__global__ __launch_bounds__(256, 2) void tree_attention_laid_kernel(TreeAttention a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char shared_lds[];
  constexpr int RB = 2 * HD, C = HD / 8, KS = HD / 32, TT = HD / 16, QH = kHalves<QT>;
  constexpr int kPlane = 32 * RB, kStage = 4 * kPlane, kPieces = 32 * C, kMine = 2 * kPieces / 256;   // (pieces: of 8 components, of the keys or the values)
  const uint32_t lds0 = (uint32_t)(uintptr_t)(pf_lds_char_t*)shared_lds;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), r = lane & 15, g = lane >> 4;
  Meeting<float> w;
  if (!find_tile<float, HD, kWhole>(a, 64 * RT, w)) return;
  if constexpr (kWhole) find_rows(static_cast<const SharedAttention&>(a), w);
  const int there = (a.counts ? held(read_uniform(a.counts + w.outer), a.tokens) : a.tokens) * (int)a.by_share.d;
  const int first = w.first + 16 * RT * wave, before = held_place(w.before);
  const bool works = first < there;
  const int blocks = w.first < there ? (w.end - w.begin + 31) >> 5 : 0;
  RunningRow<HD> row[RT];
  u32x4_t qf[RT][KS][QH];
  SeenBits<TreeAttention> bits[RT];
#pragma unroll
  for (int u = 0; u < RT; ++u) {
    row[u].clear();
    int token;
    const long long place = query_place(a, w.key_head, w.first_sequence, min(first + 16 * u + r, w.queries - 1), token);
    bits[u].ask(a, w.outer, token);
#pragma unroll
    for (int s = 0; s < KS; ++s) to_halves(load8_raw(reinterpret_cast<const QT*>(a.q) + place * HD + 32 * s + 8 * g), qf[u][s]);
  }

  // the lane's pieces of a block (past the last row: that one again)
  Raw8F32 raw[kMine];
  auto fetch = [&](int n) __attribute__((always_inline)) {
    const int at = w.begin + 32 * n, last = w.end - 1 - at;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int piece = t + 256 * i, k = min(piece % kPieces / C, last);
      raw[i] = load8_raw((piece < kPieces ? w.keys : w.values) + (size_t)at * HD + k * HD + 8 * (piece % C));
    }
  };
  auto lay_down = [&](int stage) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int piece = t + 256 * i, k = piece % kPieces / C, c = piece % C;
      const int chunk = piece < kPieces ? c ^ (k & (C - 1)) : (((c >> 1) ^ (k & (TT - 1))) << 1) | (c & 1);
      unsigned char* to = shared_lds + stage * kStage + (piece < kPieces ? 0 : 2 * kPlane) + k * RB + 16 * chunk;
      u32x4_t halves[2];
      to_halves(raw[i], halves);
      *reinterpret_cast<u32x4_t*>(to) = halves[0];
      *reinterpret_cast<u32x4_t*>(to + kPlane) = halves[1];
    }
  };
  auto lds_barrier = [] __attribute__((always_inline)) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };
  const int vkey = 4 * g + (r >> 2);
  const uint32_t k_rd = lds0 + (uint32_t)(r * RB + 16 * (g ^ (r & (C - 1))));
  const uint32_t v_rd = lds0 + (uint32_t)(2 * kPlane + vkey * RB + 32 * (vkey & (TT - 1)) + 8 * (r & 3));
  if (blocks > 0) {
    fetch(0);
    lay_down(0);
    if (blocks > 1) fetch(1);
    lds_barrier();
  }
#pragma unroll 1
  for (int n = 0; n < blocks; ++n) {
    if (n + 1 < blocks) {
      lay_down((n + 1) & 1);
      if (n + 2 < blocks) fetch(n + 2);
    }
    if (works) {
      const int at = w.begin + 32 * n;
      const uint32_t stage = (uint32_t)((n & 1) * kStage);
      f32x4_t sc[RT][2];
#pragma unroll
      for (int u = 0; u < RT; ++u) sc[u][0] = sc[u][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int kh = 0; kh < 2; ++kh) {
            const u32x4_t k = pf_read128((k_rd ^ (uint32_t)(64 * s)) + stage + (uint32_t)(kh * kPlane + jb * 16 * RB));
#pragma unroll
            for (int u = 0; u < RT; ++u)
#pragma unroll
              for (int qh = 0; qh < QH; ++qh)
                if (kh + qh < 2) sc[u][jb] = mfma16(k, qf[u][s][qh], sc[u][jb]);   // (lo times lo is beyond what is kept)
          }
      u32x4_t pf[RT];
#pragma unroll
      for (int u = 0; u < RT; ++u) {
        const int seen = w.end - at;   // of the block's rows
        if (seen < 32 || at + 32 > before) {
          const uint32_t word = ((at + 32 > before ? bits[u].of(a, at - before) : ~0u) & (seen < 32 ? (1u << max(seen, 0)) - 1u : ~0u)) >> (4 * g);
#pragma unroll
          for (int jb = 0; jb < 2; ++jb)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if ((word >> (16 * jb + i) & 1) == 0) sc[u][jb][i] = -INFINITY;
        }
        float p[8];
        to_probabilities<HD, 2>(row[u], sc[u], a.scale2, p);
        pf[u] = pack8_bf16(p);
      }
#pragma unroll
      for (int o = 0; o < TT; ++o)
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) {
          const uint32_t from = (v_rd ^ (uint32_t)(32 * o)) + stage + (uint32_t)(kh * kPlane);
          const u32x2_t lo = pf_read_tr(from), hi = pf_read_tr(from + 16 * RB);
          const u32x4_t v = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
          for (int u = 0; u < RT; ++u) row[u].o[o] = mfma16(v, pf[u], row[u].o[o]);
        }
    }
    lds_barrier();
  }

#pragma unroll
  for (int u = 0; u < RT; ++u) {
    const float l = quad_sum(row[u].l);
    const int n = first + 16 * u + r;
    if (n >= w.queries) continue;
    int token;
    query_place(a, w.key_head, w.first_sequence, n, token);
    auto put = [&](auto* to, float scale) __attribute__((always_inline)) {
#pragma unroll
      for (int o = 0; o < TT; ++o) store_run(to + 16 * o + 4 * g, row[u].o[o], scale);
    };
    if constexpr (kWhole) {
      float scale;
      uint16_t* out = result_place<HD>(a, w, n, token, l, scale);
      put(out, scale);
    } else {
      const long long place = part_place(a, w.part, w.key_head, n);
      if (g == 0) a.part_ml[place] = row[u].part(l);
      put(a.part_sums + place * HD, 1.f);
    }
  }
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
