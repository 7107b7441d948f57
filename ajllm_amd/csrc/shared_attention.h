// Attention of sequences that share a prefix: token t of sequence b sees its group's prefix rows and its own rows up to its own.
//
//   out[b, t, h] = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c q . k_j - m),  c = log2(e) / sqrt(HD),  m a number near the largest exponent
//
// The keys fall into two sets, and a softmax over both is put together from the (m, sum p, sum p v) of any parts of them.  The prefix's
// rows are met by the queries of ALL sequences of the group, as a matrix product's rows; a sequence's own rows by its own queries.
//
// Products run on bf16 MFMA, transposed so that no operand changes its layout between them (as in prefill_attention.h):
//   S^T = K Q^T    A = 16 keys x 32 dims from row-major key rows in LDS, B = queries; lane (g = l / 16, r = l % 16) gets keys 4 g .. 4 g + 3 of
//                  query r;
//   O^T += V^T P^T the lane's probabilities of 32 keys are its B fragment as they are; V^T by transposing reads of row-major rows.
// A key's 16-byte chunks (a value row's 32-byte segments) sit in slots permuted by the row, so that these reads spread over the banks.
// fp32 queries and fp32 rows are taken as two bf16 each (x = hi + lo, 16 bits): one product more for each; probabilities are
// rounded to bf16, whose 2^-9 at most a weight is what the bf16 result's own rounding is.  Everything else is fp32.
#pragma once
#include "lane_rows.h"
#include <type_traits>

#include "gemm_turns_kernels.h"  // turn_barrier
#include "prefill_attention.h"   // the fragment reads, pack8_bf16; dma16

namespace ajq {

struct SharedAttention {
  const void *q, *prefix_keys, *prefix_values, *keys, *values;
  const long long *prefix_lengths, *rows, *counts, *offset;
  uint16_t* out;
  float2* part_ml;      // [parts, queries] (m, sum p)
  float* part_sums;     // [parts, queries, HD] sum p v
  long long prefix_group, prefix_head, cache_batch, cache_head;
  long long queries;    // batch * heads * tokens, in the order of q
  int groups, batch, tokens, heads, kv_heads, prefix_cap, max_len;
  int prefix_blocks, prefix_parts, prefix_tiles, own_parts, own_tiles;
  int own_alone;        // a wave has a tile of a sequence's queries and its rows to itself, a workgroup four such
  float scale2;         // log2(e) / sqrt(HD)
  Divide by_share, by_each, by_tokens, by_heads, by_kv_heads, by_group;   // heads / kv_heads, that times tokens, .., batch / groups
  Divide by_prefix_tiles, by_prefix_parts, by_own_tiles, by_own_parts;
};

// a number that every lane of a workgroup reads, kept where such numbers are
__device__ __forceinline__ long long read_uniform(const long long* p) {
  const unsigned long long v = (unsigned long long)*p;
  return (long long)((unsigned long long)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) |
                     (unsigned long long)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32);
}
__device__ __forceinline__ int held(long long n, int most) { return (int)min(max(n, 0ll), (long long)most); }

// What a workgroup works on: a tile of the queries that meet one run of rows.
template <typename CacheT> struct Meeting {
  const CacheT *keys, *values;   // of the (group or sequence, key head)
  int key_head, first_sequence;  // the queries are those of `sequences` sequences from here on and of the key head's heads
  int queries;                   // sequences * tokens * share
  int first;                     // the tile's first query
  int part, parts, outer;        // part of the rows of sequence or group `outer`
  int begin, end;                // rows
  const CacheT *own_keys, *own_values;   // a second run of rows, from its first on (only where a workgroup walks both: `own` is then false and
  int own_end;                           // the queries are one sequence's)
  bool own, alone;               // (alone: a wave's, not a workgroup's)
  long long before;              // own rows a sequence's first new token sees ahead of its own row
};

// query number n of a meeting -> its place in q (and of its partial results), the token
__device__ __forceinline__ long long query_place(const SharedAttention& a, int key_head, int first_sequence, int n, int& token) {
  int rest, head;
  const int sequence = divide(n, a.by_each, rest);
  token = divide(rest, a.by_share, head);
  return ((long long)(first_sequence + sequence) * a.heads + (key_head * (int)a.by_share.d + head)) * a.tokens + token;
}

// 8 query components at p as bf16: hi (and lo, what fp32 has beyond it)
__device__ __forceinline__ void split8(const float* v, u32x4_t& hi, u32x4_t& lo) {
  hi = pack8_bf16(v);
  float rest[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    widen2(hi[i], a, b);
    rest[2 * i] = v[2 * i] - a;
    rest[2 * i + 1] = v[2 * i + 1] - b;
  }
  lo = pack8_bf16(rest);
}
template <typename T> constexpr int kHalves = sizeof(T) == 4 ? 2 : 1;   // bf16 numbers that stand for one
template <typename T> using Raw8 = decltype(load8_raw(static_cast<const T*>(nullptr)));
__device__ __forceinline__ void to_halves(const Raw8F32& x, u32x4_t* to) {
  const float v[8] = {x.a.x, x.a.y, x.a.z, x.a.w, x.b.x, x.b.y, x.b.z, x.b.w};
  split8(v, to[0], to[1]);
}
__device__ __forceinline__ void to_halves(const u32x4_t& x, u32x4_t* to) { to[0] = x; }

// The running softmax of 16 queries, one a lane & 15: m, the lane's own part of the sum, and HD / 16 accumulators of O^T.
template <int HD> struct RunningRow {
  f32x4_t o[HD / 16];
  float m, l;   // (m: -inf while no visible row has been met)
  // as a part's: nothing met weighs nothing, unless it was no number
  __device__ __forceinline__ float2 part(float all) const { return float2{m == -INFINITY && all != 0.f ? 0.f : m, all}; }
  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int t = 0; t < HD / 16; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
};
// Where a lane's sum of new probabilities has outgrown the reference point (or is no number: there is none yet): it moves to the largest of a query's scores if
// that is past the slack, and what has been summed up follows.  sc: N scores not scaled yet -> p and their sum.
template <int HD, int N, bool kSums>
__device__ __forceinline__ void move_point(RunningRow<HD>& row, const f32x4_t* sc, float scale2, float* p, float& sum) {
  float top = sc[0][0];
#pragma unroll
  for (int e = 1; e < N; ++e) top = fmaxf(top, sc[e >> 2][e & 3]);
  top = quad_max(top) * scale2;
  const float m = top > row.m + kPfSlack ? top : row.m;   // (nothing is more than -inf by no number)
  const float corr = m == row.m ? 1.0f : exp2_hw(row.m - m);
  sum = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    p[e] = exp2_hw(m == -INFINITY ? sc[e >> 2][e & 3] : __builtin_fmaf(sc[e >> 2][e & 3], scale2, -m));   // (0, or NaN, while there is none)
    sum += p[e];
  }
  row.m = m;
  row.l *= corr;
  if (kSums) {
#pragma unroll
    for (int t = 0; t < HD / 16; ++t) row.o[t] *= corr;
  }
}

// N 16-key tiles of scores, scaled here -> probabilities.  (The test of the sum: prefill_attention.h.)
template <int HD, int N>
__device__ __forceinline__ void to_probabilities(RunningRow<HD>& row, const f32x4_t (&sc)[N], float scale2, float (&p)[4 * N]) {
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 4 * N; ++e) {
    p[e] = exp2_hw(__builtin_fmaf(sc[e >> 2][e & 3], scale2, -row.m));
    sum += p[e];
  }
  if (__builtin_amdgcn_ballot_w64(!(sum <= kPfTrigger)) != 0) move_point<HD, 4 * N, true>(row, sc, scale2, p, sum);
  row.l += sum;
}

// A launch's workgroups: first the prefix's (a part of a (group, key head)'s rows and a tile of queries each; those that share rows are next
// to each other on one XCD), then the sequences' own likewise.  What this takes is known without the lengths on the device.
template <typename CacheT, int HD>
__device__ __forceinline__ bool find_meeting(const SharedAttention& a, int tile_queries_prefix, int tile_queries_own, Meeting<CacheT>& w) {
  w.own = (int)blockIdx.x >= a.prefix_blocks;
  w.alone = w.own && a.own_alone;
  const int id = (int)blockIdx.x - (w.own ? a.prefix_blocks : 0);
  w.parts = w.own ? a.own_parts : a.prefix_parts;
  int tile;
  const int run = w.alone ? divide(4 * id + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), a.by_own_tiles, tile)
                          : (id & 7) + 8 * divide(id >> 3, w.own ? a.by_own_tiles : a.by_prefix_tiles, tile);
  if (run >= (w.own ? a.batch : a.groups) * a.kv_heads * w.parts) return false;
  const int unit = divide(run, w.own ? a.by_own_parts : a.by_prefix_parts, w.part);
  w.outer = divide(unit, a.by_kv_heads, w.key_head);
  const int each = (int)a.by_group.d;
  w.first_sequence = w.own ? w.outer : w.outer * each;
  w.queries = (w.own ? 1 : each) * (int)a.by_each.d;
  w.first = tile * (w.own ? tile_queries_own : tile_queries_prefix);
  const size_t at = w.own ? (size_t)w.outer * a.cache_batch + (size_t)w.key_head * a.cache_head
                          : (size_t)w.outer * a.prefix_group + (size_t)w.key_head * a.prefix_head;
  w.keys = reinterpret_cast<const CacheT*>(w.own ? a.keys : a.prefix_keys) + at;
  w.values = reinterpret_cast<const CacheT*>(w.own ? a.values : a.prefix_values) + at;
  return true;
}
// Its rows: a part of whole blocks of 32.
template <typename CacheT>
__device__ __forceinline__ void find_rows(const SharedAttention& a, Meeting<CacheT>& w) {
  int rows;
  w.before = 0;
  if (w.own) {
    w.before = read_uniform(a.rows + w.outer) + (a.offset ? read_uniform(a.offset) : 0ll);
    rows = held(w.before + (a.counts ? held(read_uniform(a.counts + w.outer), a.tokens) : a.tokens), a.max_len);
  } else {
    rows = held(read_uniform(a.prefix_lengths + w.outer), a.prefix_cap);
  }
  const int per = ((rows + w.parts - 1) / w.parts + 31) & ~31;
  w.begin = (int)min((long long)rows, (long long)w.part * per);
  w.end = min(rows, w.begin + per);
}

// Both runs of one sequence's queries: its group's prefix, and its own rows.
template <int HD, typename CacheT>
__device__ __forceinline__ void find_both(const SharedAttention& a, Meeting<CacheT>& w) {
  int unused;
  const int group = divide(w.outer, a.by_group, unused);
  w.own_keys = w.keys;
  w.own_values = w.values;
  w.own = false;
  w.before = read_uniform(a.rows + w.outer) + (a.offset ? read_uniform(a.offset) : 0ll);
  w.own_end = held(w.before + (a.counts ? held(read_uniform(a.counts + w.outer), a.tokens) : a.tokens), a.max_len);
  w.begin = 0;
  w.end = held(read_uniform(a.prefix_lengths + group), a.prefix_cap);
  const size_t at = (size_t)group * a.prefix_group + (size_t)w.key_head * a.prefix_head;
  w.keys = reinterpret_cast<const CacheT*>(a.prefix_keys) + at;
  w.values = reinterpret_cast<const CacheT*>(a.prefix_values) + at;
}

// ---- Few queries: the four waves of a workgroup take blocks of 32 rows in turn, each for itself (no barrier until the end), and RT tiles of 16
// queries meet every row fetched.  Where there are sequences enough, each wave takes all rows of its own tile instead, and has nobody to join.  What bounds
// it (but for tiles of 32 on fp32 rows) is memory: a wave asks for the next block's keys as soon as it has used this block's, and for its values likewise; eight
// waves a CU (bf16) then have 64 to 128 KB on their way.  8 prompts of 1500 rows with 8 sequences of 300 each (12 heads of 64, 59 MB) 12.8 us = 4.6 TB/s.
// LDS of a wave: keys, then values, 32 rows each; fp32 rows as two planes of bf16, through registers.  Tiles of 32 queries on fp32 rows are bound by that: each wave splits its
// rows for its 32 queries alone, and one wave a SIMD (212 registers) has nothing to run beside it.  16 sequences of 100 tokens x 4 of 8 heads behind 2048 rows 386 us: 39 % of a SIMD's
// cycles are vector instructions, 16 % MFMAs.
template <int HD, typename CacheT> constexpr int few_wave_bytes() { return 2 * 32 * 2 * HD * kHalves<CacheT>; }
template <int HD, int RT> constexpr int few_join_bytes() { return 4 * RT * 16 * (HD + 4) * 4; }
template <int HD, typename CacheT, int RT> constexpr int few_lds_bytes() {
  constexpr int walk = 4 * few_wave_bytes<HD, CacheT>(), join = few_join_bytes<HD, RT>() + 4 * RT * 16 * 8;
  return walk > join ? walk : join;
}

typedef float f32x2_t __attribute__((ext_vector_type(2)));
// Components of a query's result as they are summed up, or as bf16 times scale (0: zeros, whatever they are).
__device__ __forceinline__ void store_run(float* to, f32x4_t x, float) { *reinterpret_cast<f32x4_t*>(to) = x; }
__device__ __forceinline__ void store_run(float* to, f32x2_t x, float) { *reinterpret_cast<f32x2_t*>(to) = x; }
__device__ __forceinline__ void store_run(uint16_t* to, f32x4_t x, float scale) {
  *reinterpret_cast<u32x2_t*>(to) = scale == 0.f ? u32x2_t{0u, 0u} : u32x2_t{pack2_bf16(x[0] * scale, x[1] * scale), pack2_bf16(x[2] * scale, x[3] * scale)};
}
__device__ __forceinline__ void store_run(uint16_t* to, f32x2_t x, float scale) {
  *reinterpret_cast<uint32_t*>(to) = scale == 0.f ? 0u : pack2_bf16(x[0] * scale, x[1] * scale);
}
// Where a query of a workgroup (or wave) that meets all of its rows goes, and one over its weights' sum (0 where a token is not there or saw nothing).
template <int HD, typename CacheT>
__device__ __forceinline__ uint16_t* result_place(const SharedAttention& a, const Meeting<CacheT>& w, int n, int token, float l, float& scale) {
  int rest, share;
  divide(n, a.by_each, rest);
  divide(rest, a.by_share, share);
  const bool there = a.counts == nullptr || token < a.counts[w.outer];
  scale = there && (l > 0.f || l != l) ? 1.f / l : 0.f;
  return a.out + (((size_t)w.outer * a.tokens + token) * a.heads + (w.key_head * (int)a.by_share.d + share)) * HD;
}

// A wave's results are the workgroup's (Meeting::alone).  put(u, to, scale): a lane's sums of its query of tile u, to the query's row.
template <int HD, int RT, bool kWhole, typename CacheT, typename Put>
__device__ __forceinline__ void leave_alone(const SharedAttention& a, const Meeting<CacheT>& w, const RunningRow<HD> (&row)[RT], Put put) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int u = 0; u < RT; ++u) {
    const float l = quad_sum(row[u].l);
    const int n = w.first + 16 * u + r;
    if (n >= w.queries) continue;
    int token;
    const long long in_q = query_place(a, w.key_head, w.first_sequence, n, token);
    if constexpr (kWhole) {
      float scale;
      uint16_t* out = result_place<HD>(a, w, n, token, l, scale);
      put(u, out, scale);
    } else {
      const long long place = in_q + a.prefix_parts * a.queries;
      if (g == 0) a.part_ml[place] = row[u].part(l);
      put(u, a.part_sums + place * HD, 1.f);
    }
  }
}

// The four waves' results meet in LDS (rows of HD + 4 numbers: sixteen queries' pieces fall on different banks) and become the workgroup's part, or
// (kWhole) the result.
template <int HD, int RT, int kMl, bool kWhole, typename CacheT, typename Put>
__device__ __forceinline__ void join_waves(const SharedAttention& a, const Meeting<CacheT>& w, unsigned char* lds, const RunningRow<HD> (&row)[RT], Put put) {
  constexpr int kJoin = RT * 16, kPitch = HD + 4, kHelpers = 256 / kJoin;   // queries, lanes that put one together
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  float* sums = reinterpret_cast<float*>(lds);
  float2* ml = reinterpret_cast<float2*>(lds + kMl);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < RT; ++u) {
    const float l = quad_sum(row[u].l);
    if (g == 0) ml[wave * kJoin + 16 * u + r] = row[u].part(l);
    put(u, sums + (wave * kJoin + 16 * u + r) * kPitch, 1.f);
  }
  __syncthreads();
  const int n = (int)threadIdx.x / kHelpers, d0 = 4 * ((int)threadIdx.x % kHelpers);
  if (w.first + n >= w.queries) return;
  float2 e[4];
  float m = -INFINITY, l = 0.f, weight[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    e[k] = ml[k * kJoin + n];
    m = fmaxf(m, e[k].x);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    weight[k] = e[k].x == -INFINITY ? 0.f : exp2_hw(e[k].x - m);
    l += e[k].y * weight[k];
  }
  int token;
  const long long in_q = query_place(a, w.key_head, w.first_sequence, w.first + n, token);
  const long long place = in_q + (kWhole ? 0 : (w.part + (w.own ? a.prefix_parts : 0)) * a.queries);
  if (!kWhole && d0 == 0) a.part_ml[place] = float2{m, l};
  float scale = 1.f;
  uint16_t* out = nullptr;
  if constexpr (kWhole) out = result_place<HD>(a, w, w.first + n, token, l, scale);
#pragma unroll
  for (int d = 0; d < HD; d += 4 * kHelpers) {
    if (d + d0 >= HD) break;
    f32x4_t o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) o += *reinterpret_cast<const f32x4_t*>(sums + (k * kJoin + n) * kPitch + d + d0) * weight[k];
    if constexpr (kWhole) store_run(out + d + d0, o, scale);
    else store_run(a.part_sums + place * HD + d + d0, o, 1.f);
  }
}

// Block n (of N rows) of a meeting's rows: of the second run's behind the first's (kBoth).
template <int HD, int N, bool kBoth, typename CacheT> struct Block {
  const CacheT *keys, *values;   // its first row
  int rows;                      // from there on in its run
  int at;                        // its first row's number there
  bool second;
  __device__ __forceinline__ Block(const Meeting<CacheT>& w, int n) {
    const int of_first = (w.end - w.begin + N - 1) / N;
    second = kBoth && n >= of_first;
    at = second ? N * (n - of_first) : w.begin + N * n;
    rows = (second ? w.own_end : w.end) - at;
    keys = (second ? w.own_keys : w.keys) + (size_t)at * HD;
    values = (second ? w.own_values : w.values) + (size_t)at * HD;
  }
};
template <int N, bool kBoth, typename CacheT>
__device__ __forceinline__ int blocks_of(const Meeting<CacheT>& w) {
  return (w.end - w.begin + N - 1) / N + (kBoth ? (w.own_end + N - 1) / N : 0);
}

// W: how many of the waves work.
template <int HD, typename QT, typename CacheT, int RT, int W = 4, bool kBoth = false>
__device__ __forceinline__ void meet_few(const SharedAttention& a, Meeting<CacheT>& w, unsigned char* lds, uint32_t lds0) {
  constexpr int RB = 2 * HD, C = HD / 8, KS = HD / 32, TT = HD / 16, KH = kHalves<CacheT>, QH = kHalves<QT>;
  constexpr int kPlane = 32 * RB;                 // 32 rows of bf16
  constexpr bool kDma = KH == 1;
  constexpr int kRows = 1024 / RB;                // rows of one wave-wide request
  constexpr int kAsk = 32 / kRows;                // requests a block of keys (or values)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t mine = lds0 + (uint32_t)(wave * few_wave_bytes<HD, CacheT>());
  unsigned char* mine_p = lds + wave * few_wave_bytes<HD, CacheT>();

  // ---- queries: fragments of RT tiles (asked for ahead of the lengths, of which nothing in them depends)
  Raw8<QT> raw[RT][KS];
  int token[RT];
#pragma unroll
  for (int u = 0; u < RT; ++u) {
    const long long place = query_place(a, w.key_head, w.first_sequence, min(w.first + 16 * u + r, w.queries - 1), token[u]);
#pragma unroll
    for (int s = 0; s < KS; ++s) raw[u][s] = load8_raw(reinterpret_cast<const QT*>(a.q) + place * HD + 32 * s + 8 * g);
  }
  __builtin_amdgcn_sched_barrier(0);
  kBoth ? find_both<HD>(a, w) : find_rows(a, w);
  RunningRow<HD> row[RT];
  int limit[RT];   // how many of the meeting's rows (kBoth: of the second run's) a lane's queries see
#pragma unroll
  for (int u = 0; u < RT; ++u) {
    limit[u] = kBoth ? held(w.before + token[u] + 1, w.own_end) : w.own ? held(w.before + token[u] + 1, w.end) : w.end;
    row[u].clear();
  }

  // ---- rows on their way (past the last: the last again, which is there and finite)
  const int ask_row = lane / C, slot = lane % C;
  using Rows = Block<HD, 32, kBoth, CacheT>;
  auto ask = [&](const CacheT* from, int rows, uint32_t to, bool values) {
#pragma unroll
    for (int i = 0; i < kAsk; ++i) {
      const int k = kRows * i + ask_row;
      const uint32_t chunk = values ? (uint32_t)((((slot >> 1) ^ (k & (TT - 1))) << 1) | (slot & 1)) : (uint32_t)(slot ^ (k & (C - 1)));
      dma16(from, (uint32_t)(min(k, rows - 1) * RB) + chunk * 16u, to + (uint32_t)(i * 1024));
    }
  };
  constexpr int kPieces = kDma ? 1 : 32 * C / 64;   // 8 components each, a lane
  Raw8F32 kraw[kPieces], vraw[kPieces];
  auto fetch = [&](const Rows& from) {
    if constexpr (!kDma) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int piece = lane + 64 * i, k = min(piece / C, from.rows - 1);
        kraw[i] = load8_raw(from.keys + k * HD + 8 * (piece % C));
        vraw[i] = load8_raw(from.values + k * HD + 8 * (piece % C));
      }
    }
  };
  auto lay_down = [&]() {
    if constexpr (!kDma) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int piece = lane + 64 * i, k = piece / C, c = piece % C;
        auto put = [&](const Raw8F32& x, unsigned char* to) {
          u32x4_t halves[2];
          to_halves(x, halves);
          *reinterpret_cast<u32x4_t*>(to) = halves[0];
          *reinterpret_cast<u32x4_t*>(to + kPlane) = halves[1];
        };
        put(kraw[i], mine_p + k * RB + 16 * (c ^ (k & (C - 1))));
        put(vraw[i], mine_p + 2 * kPlane + k * RB + 16 * ((((c >> 1) ^ (k & (TT - 1))) << 1) | (c & 1)));
      }
    }
  };
  const uint32_t values0 = mine + (uint32_t)(KH * kPlane);
  uint32_t k_rd[KS], v_rd[TT];
#pragma unroll
  for (int s = 0; s < KS; ++s) k_rd[s] = mine + (uint32_t)(r * RB + 16 * ((4 * s + g) ^ (r & (C - 1))));
  const int vkey = 4 * g + (r >> 2);
#pragma unroll
  for (int t = 0; t < TT; ++t) v_rd[t] = values0 + (uint32_t)(vkey * RB + 32 * (t ^ (vkey & (TT - 1))) + 8 * (r & 3));

  const int blocks = w.alone || wave < W ? blocks_of<32, kBoth>(w) : 0, begin = w.alone ? 0 : wave, by = w.alone ? 1 : W;
  if (begin < blocks) {
    const Rows first(w, begin);
    if constexpr (kDma) {
      ask(first.keys, first.rows, mine, false);
      ask(first.values, first.rows, values0, true);
    } else {
      fetch(first);
    }
  }
  u32x4_t qf[RT][KS][QH];
#pragma unroll
  for (int u = 0; u < RT; ++u)
#pragma unroll
    for (int s = 0; s < KS; ++s) to_halves(raw[u][s], qf[u][s]);
  for (int n = begin; n < blocks; n += by) {
    const bool more = n + by < blocks;
    const Rows now(w, n), next(w, more ? n + by : n);
    if constexpr (kDma) {
      // (behind this block's keys only its values are on their way)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kAsk) : "memory");
    } else {
      lay_down();
      if (more) fetch(next);
      wave_lds_order();
    }
    f32x4_t sc[RT][2];
#pragma unroll
    for (int u = 0; u < RT; ++u) sc[u][0] = sc[u][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
#pragma unroll
      for (int jb = 0; jb < 2; ++jb) {
#pragma unroll
        for (int kh = 0; kh < KH; ++kh) {
          const u32x4_t k = pf_read128(k_rd[s] + (uint32_t)(kh * kPlane + jb * 16 * RB));
#pragma unroll
          for (int u = 0; u < RT; ++u)
#pragma unroll
            for (int qh = 0; qh < QH; ++qh)
              if (kh + qh < 2) sc[u][jb] = mfma16(k, qf[u][s][qh], sc[u][jb]);   // (lo times lo is beyond what is kept)
        }
      }
    }
    if constexpr (kDma) {
      if (more) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        ask(next.keys, next.rows, mine, false);
      }
    }
    u32x4_t pf[RT];
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      const int seen = (kBoth && !now.second ? w.end : limit[u]) - now.at;   // of the block's rows
      if (__builtin_amdgcn_ballot_w64(seen < 32) != 0) {
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * jb + 4 * g + i >= seen) sc[u][jb][i] = -INFINITY;
      }
      float p[8];
      to_probabilities<HD, 2>(row[u], sc[u], a.scale2, p);
      pf[u] = pack8_bf16(p);
    }
    if constexpr (kDma) {
      if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kAsk) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
#pragma unroll
    for (int t = 0; t < TT; ++t) {
#pragma unroll
      for (int kh = 0; kh < KH; ++kh) {
        const u32x2_t lo = pf_read_tr(v_rd[t] + (uint32_t)(kh * kPlane)), hi = pf_read_tr(v_rd[t] + (uint32_t)(kh * kPlane + 16 * RB));
        const u32x4_t v = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
        for (int u = 0; u < RT; ++u) row[u].o[t] = mfma16(v, pf[u], row[u].o[t]);
      }
    }
    if constexpr (kDma) {
      if (more) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        ask(next.values, next.rows, values0, true);
      }
    } else {
      wave_lds_order();
    }
  }

  auto put = [&](int u, auto* to, float scale) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < TT; ++t) store_run(to + 16 * t + 4 * g, row[u].o[t], scale);
  };
  if (w.alone) leave_alone<HD, RT, kBoth>(a, w, row, put);
  else join_waves<HD, RT, few_join_bytes<HD, RT>(), kBoth>(a, w, lds, row, put);
}

// ---- At most 16 queries on fp32 rows, in fp32 throughout (v_mfma_f32_16x16x4_f32: 32 cycles for 16 rows x 4 components, where the memory's share of a CU
// brings them in more).  Rows go from memory to registers as the products take them; nothing passes LDS.  A wave takes 16 rows at a time.
//   S^T: lane (g, r) holds components 16 c + 4 g .. + 3 of key r and of query r; step (c, e) multiplies the e-th of each.
//   O^T: lane (g, r) has the weights of keys 4 g .. 4 g + 3; step i takes key 4 g + i and, of its values, components P r .. P r + P - 1 of every
//   16 P (P = 4, or 2 where there are 32): tile (v, e) is then components 16 P v + P m + e, m = 0 .. 15.
__device__ __forceinline__ float4 query4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 query4(const uint16_t* p) {
  const u32x2_t w = *reinterpret_cast<const u32x2_t*>(p);
  float4 v;
  widen2(w.x, v.x, v.y);
  widen2(w.y, v.z, v.w);
  return v;
}
template <int HD> constexpr int few_f32_lds_bytes() { return few_join_bytes<HD, 1>() + 4 * 16 * 8; }
template <int HD, typename QT, bool kBoth = false>
__device__ __forceinline__ void meet_few_f32(const SharedAttention& a, Meeting<float>& w, unsigned char* lds) {
  constexpr int KC = HD / 16, P = HD == 32 ? 2 : 4, VC = HD / (16 * P);
  typedef float part_t __attribute__((ext_vector_type(P)));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  int token;
  const QT* from = reinterpret_cast<const QT*>(a.q) + query_place(a, w.key_head, w.first_sequence, min(w.first + r, w.queries - 1), token) * HD + 4 * g;
  float4 q[KC];
#pragma unroll
  for (int c = 0; c < KC; ++c) q[c] = query4(from + 16 * c);
  __builtin_amdgcn_sched_barrier(0);
  kBoth ? find_both<HD>(a, w) : find_rows(a, w);
  const int limit = kBoth ? held(w.before + token + 1, w.own_end) : w.own ? held(w.before + token + 1, w.end) : w.end;
  using Rows = Block<HD, 16, kBoth, float>;
  RunningRow<HD> row[1];
  row[0].clear();
  struct Fetched {
    float4 k[KC];
    part_t v[4][VC];
  };
  auto ask = [&](const Rows& from, Fetched& to) __attribute__((always_inline)) {   // (past the last row: that one again)
    const float* keys = from.keys + min(r, from.rows - 1) * HD + 4 * g;
#pragma unroll
    for (int c = 0; c < KC; ++c) to.k[c] = *reinterpret_cast<const float4*>(keys + 16 * c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* values = from.values + min(4 * g + i, from.rows - 1) * HD + P * r;
#pragma unroll
      for (int c = 0; c < VC; ++c) to.v[i][c] = *reinterpret_cast<const part_t*>(values + 16 * P * c);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto meet = [&](int n, const Fetched& rows) __attribute__((always_inline)) {
    const Rows now(w, n);
    const int seen = (kBoth && !now.second ? w.end : limit) - now.at;   // of the block's rows
    f32x4_t even = f32x4_t{0.f, 0.f, 0.f, 0.f}, odd = even;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      even = __builtin_amdgcn_mfma_f32_16x16x4f32(rows.k[c].x, q[c].x, even, 0, 0, 0);
      odd = __builtin_amdgcn_mfma_f32_16x16x4f32(rows.k[c].y, q[c].y, odd, 0, 0, 0);
      even = __builtin_amdgcn_mfma_f32_16x16x4f32(rows.k[c].z, q[c].z, even, 0, 0, 0);
      odd = __builtin_amdgcn_mfma_f32_16x16x4f32(rows.k[c].w, q[c].w, odd, 0, 0, 0);
    }
    f32x4_t sc[1] = {even + odd};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * g + i >= seen) sc[0][i] = -INFINITY;
    float p[4];
    to_probabilities<HD, 1>(row[0], sc, a.scale2, p);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < VC; ++c)
#pragma unroll
        for (int e = 0; e < P; ++e) row[0].o[c * P + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(rows.v[i][c][e], p[i], row[0].o[c * P + e], 0, 0, 0);
  };
  // two blocks' registers in turn, the next one's rows on their way while one is worked on
  const int blocks = blocks_of<16, kBoth>(w), begin = w.alone ? 0 : wave, by = w.alone ? 1 : 4;
  Fetched even_rows, odd_rows;
  if (begin < blocks) ask(Rows(w, begin), even_rows);
  for (int n = begin; n < blocks; n += 2 * by) {
    if (n + by < blocks) ask(Rows(w, n + by), odd_rows);
    meet(n, even_rows);
    if (n + by >= blocks) break;
    if (n + 2 * by < blocks) ask(Rows(w, n + 2 * by), even_rows);
    meet(n + by, odd_rows);
  }
  // a lane has components 16 P v + P (4 g + i) + e of query r: of each v 4 P of them one behind the other
  auto put = [&](int, auto* to, float scale) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        part_t x;
#pragma unroll
        for (int e = 0; e < P; ++e) x[e] = row[0].o[c * P + e][i];
        store_run(to + 16 * P * c + P * (4 * g + i), x, scale);
      }
  };
  if (w.alone) leave_alone<HD, 1, kBoth>(a, w, row, put);
  else join_waves<HD, 1, few_join_bytes<HD, 1>(), kBoth>(a, w, lds, row, put);
}

// ---- Many queries on bf16 rows: 64 U to a workgroup, 16 U to each wave, all four walking the same blocks of 64 rows (LDS, two stages of a key and a
// value tile, one barrier a block).  Bound by what a wave issues beside its MFMAs.  The walk goes over a run of the group's prefix and, behind it, of one sequence's own
// rows; either may be empty.  It goes in steps of 32 rows; step t holds the exponents of step t + 1, the softmax of step t and the values of step t - 1
// times their probabilities, laid out in HD / 16 pieces of either product with their share of the exponentials, in that order for good, so that a
// wave has MFMAs and vector work to issue side by side (attn_prefill_steps_kernel).
//
// Keys of block j + 2 and values of block j + 1 are asked for in the second step of block j.  A prefix that few tiles of queries walk at a time comes from
// HBM, whose latency is longer than a block: the lines of block j + 4 are touched then as well (four bytes each, into a corner of
// LDS that nobody reads), so that the requests themselves find them in L2.
template <typename CacheT> struct Walk {
  const CacheT *keys[2], *values[2];   // the part's first rows: prefix, own
  int rows[2];                         // how many there are
  int key_head, first_sequence, queries, first;
  long long before;                    // own rows ahead of a sequence's first new token, counted from the part's first own row
};
template <int HD> constexpr int many_lds_bytes() { return 4 * 64 * 2 * HD + 4 * 256; }

// Two requests of 1 KiB each for 4096 bytes ahead of lds_addr (from 4096 bytes ahead of base) and for lds_addr: the instruction's offset moves both sides.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0, as dma16)
__device__ __forceinline__ void dma16_pair(const void* base, uint32_t voff, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:-4096\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds_addr), "v"(voff), "s"(base)
               : "memory", "m0");
}
#pragma clang diagnostic pop

template <int HD, typename QT, int U>
__device__ __forceinline__ void meet_many(const SharedAttention& a, const Walk<uint16_t>& w, RunningRow<HD> (&row)[U], uint32_t lds0) {
  constexpr int RB = 2 * HD, C = HD / 8, KS = HD / 32, TT = HD / 16, QH = kHalves<QT>, kAhead = TT < 3 ? TT : 3;
  constexpr int kTile = 64 * RB;
  constexpr int kReqRows = 1024 / RB;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    row[u].clear();
  }
  const int prefix_blocks = (w.rows[0] + 63) >> 6, blocks = prefix_blocks + ((w.rows[1] + 63) >> 6);
  if (blocks == 0) return;

  // ---- requests: 1 KiB of rows each; wave w takes rows kReqRows w .. of every group of 4 kReqRows.  Rows past a run's last: that one again.
  const int krow = kReqRows * wave + lane / C, slot = lane % C;
  const uint32_t k_lane = (uint32_t)(krow * RB) + (uint32_t)(slot ^ (krow & (C - 1))) * 16u;
  const uint32_t v_lane = (uint32_t)(krow * RB) + (uint32_t)((((slot >> 1) ^ (krow & (TT - 1))) << 1) | (slot & 1)) * 16u;
  auto place = [&](bool values, int i, int stage) __attribute__((always_inline)) {
    return lds0 + (uint32_t)(stage * 2 * kTile + (values ? kTile : 0) + (wave + 4 * i) * 1024);
  };
  auto request = [&](int j, bool values) __attribute__((always_inline)) {
    const bool own = j >= prefix_blocks;
    const int at = 64 * (own ? j - prefix_blocks : j), there = own ? w.rows[1] : w.rows[0];
    const uint16_t* from = (values ? (own ? w.values[1] : w.values[0]) : (own ? w.keys[1] : w.keys[0])) + (size_t)at * HD;
    int l = lane;   // (formed again from the lane's number: no register of its own beside the steps)
    asm volatile("" : "+v"(l));
    const int row = kReqRows * wave + l / C, to = l % C;
    const uint32_t chunk = values ? (uint32_t)((((to >> 1) ^ (row & (TT - 1))) << 1) | (to & 1)) * 16u : (uint32_t)(to ^ (row & (C - 1))) * 16u;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const uint32_t k = (uint32_t)min(4 * kReqRows * i + row, there - 1 - at) * (uint32_t)RB;
      dma16(from, k + chunk, place(values, i, j & 1));
    }
  };
  // fragments in stage 0: k-step s at k_rd ^ 64 s, output tile t at v_rd ^ 32 t.  (The body keeps all of them; the steps that go one by one have no registers
  // left for that: one that goes to memory there waits, with the memory's order, for every row on its way.)
  const int vkey = 4 * g + (r >> 2);
  const uint32_t k_rd = lds0 + (uint32_t)(r * RB + 16 * (g ^ (r & (C - 1))));
  const uint32_t v_rd = lds0 + (uint32_t)(kTile + vkey * RB + 32 * (vkey & (TT - 1)) + 8 * (r & 3));

  request(0, false);
  request(0, true);
  u32x4_t qf[U][KS][QH];
  // own rows that query n of the walk sees
  auto limit_of = [&](int n) __attribute__((always_inline)) {
    int rest, unused;
    divide(min(n, w.queries - 1), a.by_each, rest);
    return held(w.before + divide(rest, a.by_share, unused) + 1, w.rows[1]);
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    int token;
    const long long at = query_place(a, w.key_head, w.first_sequence, min(w.first + 16 * (U * wave + u) + r, w.queries - 1), token);
#pragma unroll
    for (int s = 0; s < KS; ++s) to_halves(load8_raw(reinterpret_cast<const QT*>(a.q) + at * HD + 32 * s + 8 * g), qf[u][s]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int h = 0; h < QH; ++h) asm volatile("" : "+v"(qf[u][s][h]));
  const int nearest = limit_of(w.first + 16 * U * wave), farthest = limit_of(w.first + 16 * U * wave + 16 * U - 1);   // of the wave's queries
  // steps of this wave
  const int steps = w.first + 16 * U * wave >= w.queries ? 0 : farthest > 0 ? 2 * prefix_blocks + ((farthest + 31) >> 5) : (w.rows[0] + 31) >> 5;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (blocks > 1) request(1, false);
  turn_barrier();

  f32x4_t sn[U][2];  // products of the step ahead
  u32x4_t pf[U];     // probabilities of the step behind
  auto key_frag = [&](uint32_t base, int at, int i) __attribute__((always_inline)) {
    return pf_read128((base ^ (uint32_t)(64 * (i >> 1))) + (uint32_t)(at + (i & 1) * 16 * RB));
  };
  auto score = [&](const u32x4_t& kf, int i) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < QH; ++h)
#pragma unroll
      for (int u = 0; u < U; ++u) sn[u][i & 1] = mfma16(kf, qf[u][i >> 1][h], i < 2 && h == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : sn[u][i & 1]);
  };
  // Step t: products from the keys at k_at, values at v_at (kV: not in the very first), and req(piece)
  auto step = [&](int t, auto values, auto masked, int k_at, int v_at, auto req) __attribute__((always_inline)) {
    constexpr bool kV = decltype(values)::value;
    constexpr int ahead = decltype(masked)::value ? 1 : kAhead;   // (the steps that go one by one have no registers for more)
    f32x4_t sc[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int jb = 0; jb < 2; ++jb) sc[u][jb] = sn[u][jb];
    u32x4_t kf[TT];
    u32x2_t vl[TT], vh[TT];
    uint32_t k_base = k_rd, v_base = v_rd;
    if (decltype(masked)::value) asm volatile("" : "+v"(k_base), "+v"(v_base));
    auto fetch = [&](int i) __attribute__((always_inline)) {
      if (kV) {   // (first: what waits for the keys then waits for them too)
        vl[i] = pf_read_tr((v_base ^ (uint32_t)(32 * i)) + (uint32_t)v_at);
        vh[i] = pf_read_tr((v_base ^ (uint32_t)(32 * i)) + (uint32_t)(v_at + 16 * RB));
      }
      kf[i] = key_frag(k_base, k_at, i);
    };
#pragma unroll
    for (int i = 0; i < ahead; ++i) fetch(i);
    if (decltype(masked)::value) {
      const bool own = (t >> 1) >= prefix_blocks;
      const int at = 32 * (t - (own ? 2 * prefix_blocks : 0));
      if (at + 32 > (own ? nearest : w.rows[0])) {
        int l = lane;
        asm volatile("" : "+v"(l));
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int last = (own ? limit_of(w.first + 16 * (U * wave + u) + (l & 15)) : w.rows[0]) - at - 4 * (l >> 4);
#pragma unroll
          for (int jb = 0; jb < 2; ++jb)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (16 * jb + i >= last) sc[u][jb][i] = -INFINITY;
        }
      }
    }
    u32x4_t pn[U];
    float p[U][8], psum[U];
    // exponentials of a piece: beside their exponents of the next piece's and the sum of the last one's, so that none waits for what is just being made
    constexpr int kPer = 8 * U / TT;
    auto exponent = [&](int n) __attribute__((always_inline)) { return __builtin_fmaf(sc[n >> 3][(n & 7) >> 2][n & 3], a.scale2, -row[n >> 3].m); };
    auto add = [&](int n) __attribute__((always_inline)) { psum[n >> 3] = (n & 7) == 0 ? p[n >> 3][0] : psum[n >> 3] + p[n >> 3][n & 7]; };
#pragma unroll
    for (int x = 0; x < kPer; ++x) p[x >> 3][x & 7] = exponent(x);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      if (i + ahead < TT) fetch(i + ahead);
      req(i);
      score(kf[i], i);
#pragma unroll
      for (int x = 0; x < kPer; ++x) {
        const int n = i * kPer + x, u = n >> 3, e = n & 7;
        p[u][e] = exp2_hw(p[u][e]);
        if (n + kPer < 8 * U) p[(n + kPer) >> 3][(n + kPer) & 7] = exponent(n + kPer);
        if (i > 0) add(n - kPer);
        if (i == TT - 1) add(n);
      }
      if (U * (i + 1) % TT == 0) {  // a group of rows is through (pinned: the compiler would sink it behind the branches below)
        const int u = U * i / TT;
        pn[u] = pack8_bf16(p[u]);
        asm volatile("" : "+v"(pn[u]));
        if (i == TT - 1)
#pragma unroll
          for (int v = 0; v < U; ++v) asm volatile("" : "+v"(psum[v]));
      }
      if (kV) {
        const u32x4_t vf = {vl[i].x, vl[i].y, vh[i].x, vh[i].y};
#pragma unroll
        for (int u = 0; u < U; ++u) row[u].o[i] = mfma16(vf, pf[u], row[u].o[i]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (__builtin_amdgcn_ballot_w64(!(psum[u] <= kPfTrigger)) != 0) {
        move_point<HD, 8, kV>(row[u], sc[u], a.scale2, p[u], psum[u]);
        pn[u] = pack8_bf16(p[u]);
      }
      row[u].l += psum[u];
      pf[u] = pn[u];
    }
  };
  auto last_values = [&](int v_at) __attribute__((always_inline)) {
    u32x2_t vl[TT], vh[TT];
    uint32_t v_base = v_rd;
    asm volatile("" : "+v"(v_base));
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      vl[i] = pf_read_tr((v_base ^ (uint32_t)(32 * i)) + (uint32_t)v_at);
      vh[i] = pf_read_tr((v_base ^ (uint32_t)(32 * i)) + (uint32_t)(v_at + 16 * RB));
    }
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      const u32x4_t vf = {vl[i].x, vl[i].y, vh[i].x, vh[i].y};
#pragma unroll
      for (int u = 0; u < U; ++u) row[u].o[i] = mfma16(vf, pf[u], row[u].o[i]);
    }
  };
  constexpr std::integral_constant<bool, true> yes{};
  constexpr std::integral_constant<bool, false> no{};
  auto none = [](int) {};
  if (steps > 0) {
    u32x4_t kf[TT];
#pragma unroll
    for (int i = 0; i < TT; ++i) kf[i] = key_frag(k_rd, 0, i);
#pragma unroll
    for (int i = 0; i < TT; ++i) score(kf[i], i);
    step(0, no, yes, 32 * RB, 0, none);
  }
  // Blocks j (even) and j + 1 of a run at places known to the compiler: the second step of j, both of j + 1, the first of j + 2, while what they ask for and
  // multiply is whole blocks that all of the wave's queries see.  The others one by one.
  // (Two tiles of queries leave no registers to do so with the second run's: its steps all go one by one.)
  constexpr int kRuns = U == 1 ? 2 : 1;
  int t = 1;
#pragma unroll 1
  for (int run = 0; run < kRuns; ++run) {
    int j = t >> 1;
    const int ahead_of_run = run ? prefix_blocks : 0, whole = (run ? w.rows[1] : w.rows[0]) >> 6;
    const int last = min(ahead_of_run + min(whole - 4, run ? ((nearest - 32) >> 6) - 2 : whole), (steps - 6) >> 1);   // the last such j
    if (j <= last) {
      const char* const keys = reinterpret_cast<const char*>(run ? w.keys[1] : w.keys[0]);
      const char* const values = reinterpret_cast<const char*>(run ? w.values[1] : w.values[0]);
      const char* k_from = keys + (size_t)(j - ahead_of_run + 2) * kTile;
      const char* v_from = values + (size_t)(j - ahead_of_run + 1) * kTile;
      // lines: of the keys waves 0 and 1, of the values 2 and 3, of block j + 4 (of the last whole one, at most)
      const uint32_t corner = lds0 + (uint32_t)(4 * kTile + 256 * wave);
      const uint32_t line = (uint32_t)((64 * (wave & 1) + lane) * (RB / 2));
      auto touch = [&](int block) __attribute__((always_inline)) {
        dma4((wave < 2 ? keys : values) + (size_t)min(block - ahead_of_run, whole - 1) * kTile, line, corner);
      };
      touch(j + 4);
      do {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          asm volatile("s_waitcnt vmcnt(1)" ::: "memory");   // (all but the touch)
          turn_barrier();
          step(2 * j + 2 * x + 1, yes, no, (x ^ 1) * 2 * kTile, x * 2 * kTile, [&](int i) __attribute__((always_inline)) {
            const int n = i % KS;   // request of the wave: of the keys', then of the values'
            const char* const from = (i < KS ? k_from : v_from) + n * 4096;
            const uint32_t at = i < KS ? k_lane : v_lane, to = place(i >= KS, n, i < KS ? x : x ^ 1);
            if (KS == 1) dma16(from, at, to);
            else if (n % 2 == 0) dma16_pair(from + 4096, at, to + 4096);
            if (i == TT - 1) touch(j + x + 5);
          });
          k_from += kTile;
          v_from += kTile;
          step(2 * j + 2 * x + 2, yes, no, (x ^ 1) * 2 * kTile + 32 * RB, x * 2 * kTile + 32 * RB, none);
        }
        j += 2;
      } while (j <= last);
    }
    // (the first run's up to where the second's whole blocks may begin, at an even block)
    const int until = run + 1 == kRuns ? 2 * blocks : min(2 * blocks, 2 * max(j, (prefix_blocks + 1) & ~1) + 1);
    for (t = 2 * j + 1; t < until; ++t) {
      const int block = t >> 1;
      if (t & 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        turn_barrier();
        if (block + 2 < blocks) request(block + 2, false);
        if (block + 1 < blocks) request(block + 1, true);
      }
      auto half = [&](int n) { return ((n >> 1) & 1) * 2 * kTile + (n & 1) * 32 * RB; };  // where step n's keys (values) lie
      // (the last step's products of the one behind it are of no use, whatever lies there)
      if (t < steps) step(t, yes, yes, half(t + 1), half(t - 1), none);
      else if (t == steps) last_values(half(t - 1));
    }
  }
  if (steps == 2 * blocks) last_values(((blocks - 1) & 1) * 2 * kTile + 32 * RB);
}

// a lane's queries of meet_many as partial results
template <int HD, int U>
__device__ __forceinline__ void leave_part(const SharedAttention& a, const Walk<uint16_t>& w, const RunningRow<HD> (&row)[U], int part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float l = quad_sum(row[u].l);
    const int n = w.first + 16 * (U * wave + u) + r;
    if (n >= w.queries) continue;
    int token;
    const long long place = query_place(a, w.key_head, w.first_sequence, n, token) + part * a.queries;
    if (g == 0) a.part_ml[place] = row[u].part(l);
#pragma unroll
    for (int t = 0; t < HD / 16; ++t) *reinterpret_cast<f32x4_t*>(a.part_sums + place * HD + 16 * t + 4 * g) = row[u].o[t];
  }
}

template <int HD, typename QT, typename CacheT, int RT, bool kBoth = false>
__device__ __forceinline__ void meet_some(const SharedAttention& a, Meeting<CacheT>& w, unsigned char* lds, uint32_t lds0) {
  if constexpr (sizeof(CacheT) == 4 && RT == 1) meet_few_f32<HD, QT, kBoth>(a, w, lds);
  else meet_few<HD, QT, CacheT, RT, 4, kBoth>(a, w, lds, lds0);
}
template <int HD, typename CacheT, int RT> constexpr int some_lds_bytes() {
  return sizeof(CacheT) == 4 && RT == 1 ? few_f32_lds_bytes<HD>() : few_lds_bytes<HD, CacheT, RT>();
}
template <int HD, typename QT, typename CacheT, int RTP, int RTO>
__global__ __launch_bounds__(256, sizeof(CacheT) == 4 && RTP == 2 ? 1 : 2) void shared_attention_few_kernel(SharedAttention a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char shared_lds[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(pf_lds_char_t*)shared_lds;
  Meeting<CacheT> w;
  if (!find_meeting<CacheT, HD>(a, 16 * RTP, 16 * RTO, w)) return;
  if (RTP == RTO || !w.own) meet_some<HD, QT, CacheT, RTP>(a, w, shared_lds, lds0);
  else meet_some<HD, QT, CacheT, RTO>(a, w, shared_lds, lds0);
}

// Few rows in all: a workgroup walks the prefix and then a sequence's own rows with that sequence's queries alone, and what comes out is the result, in
// one launch.  Each sequence reads the prefix again (from L2), which two launches cost more than.
template <int HD, typename QT, typename CacheT>
__global__ __launch_bounds__(256, 2) void shared_attention_each_kernel(SharedAttention a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char shared_lds[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(pf_lds_char_t*)shared_lds;
  Meeting<CacheT> w;
  if (!find_meeting<CacheT, HD>(a, 16, 16, w)) return;
  meet_some<HD, QT, CacheT, 1, true>(a, w, shared_lds, lds0);
}

// The prefix by meet_many, the sequences' own rows by meet_few: beside a long prefix (U 2) by two waves a workgroup, which leave more of the memory to the prefix
// (128 sequences of 8 heads x 4 behind 32768 rows with 1000, 399 MB and 70 GFLOP, 110 us; by one wave 118, by four 115; the prefix alone 82 us = 850 TFLOP/s, own rows
// alone 55).
template <int HD, typename QT, int U>
__global__ __launch_bounds__(256, 2) void shared_attention_many_kernel(SharedAttention a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char shared_lds[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(pf_lds_char_t*)shared_lds;
  Meeting<uint16_t> w;
  if (!find_meeting<uint16_t, HD>(a, 64 * U, 16, w)) return;
  if (w.own) {
    meet_few<HD, QT, uint16_t, 1, U == 2 ? 2 : 4>(a, w, shared_lds, lds0);
    return;
  }
  find_rows(a, w);
  Walk<uint16_t> walk;
  walk.keys[0] = w.keys + (size_t)w.begin * HD;
  walk.values[0] = w.values + (size_t)w.begin * HD;
  walk.keys[1] = walk.values[1] = nullptr;
  walk.rows[0] = w.end - w.begin;
  walk.rows[1] = 0;
  walk.key_head = w.key_head;
  walk.first_sequence = w.first_sequence;
  walk.queries = w.queries;
  walk.first = w.first;
  walk.before = 0;
  RunningRow<HD> row[U];
  meet_many<HD, QT, U>(a, walk, row, lds0);
  leave_part<HD, U>(a, walk, row, w.part);
}

// Sequences with many new tokens each: 64 U queries of one sequence walk the prefix and then its own rows, and what comes out is the result.  With
// own_parts > 1 the walk is cut up and leaves parts for the merge.  16 sequences of 100 tokens x 4 of 8 heads behind 2048 rows 66 us = 630 TFLOP/s (71 in the first calls after
// a pause), 24 of 50 behind 8000 203 us = 775.  Of the former's cycles a CU is busy for 63 % (358 tiles on 256 CUs: some have two, some one), and a SIMD for 45 % of those with MFMAs,
// 36 % with other vector instructions; its LDS is no limit (no bank conflicts).
template <int HD, typename QT, int U>
__global__ __launch_bounds__(256, 2) void shared_attention_walk_kernel(SharedAttention a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char shared_lds[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(pf_lds_char_t*)shared_lds;
  const int share = (int)a.by_share.d, parts = a.own_parts;
  int part, hk, unused, tile;
  const int id = (int)blockIdx.x, run = (id & 7) + 8 * divide(divide(id >> 3, a.by_own_parts, part), a.by_own_tiles, tile);
  if (run >= a.batch * a.kv_heads) return;
  tile = a.own_tiles - 1 - tile;
  const int b = divide(run, a.by_kv_heads, hk), group = divide(b, a.by_group, unused);
  Walk<uint16_t> w;
  w.key_head = hk;
  w.first_sequence = b;
  w.queries = a.tokens * share;
  w.first = 64 * U * tile;
  w.before = read_uniform(a.rows + b) + (a.offset ? read_uniform(a.offset) : 0ll);
  const int there = a.counts ? held(read_uniform(a.counts + b), a.tokens) : a.tokens;
  const int last = min(divide(w.first + 64 * U - 1, a.by_share, unused), there - 1);          // the tile's last token that is there
  const size_t at = (size_t)group * a.prefix_group + (size_t)hk * a.prefix_head, own = (size_t)b * a.cache_batch + (size_t)hk * a.cache_head;
  const bool none = w.first >= there * share;
  const int prefix_rows = none ? 0 : held(read_uniform(a.prefix_lengths + group), a.prefix_cap), own_rows = none ? 0 : held(w.before + last + 1, a.max_len);
  // this part's blocks: first .. first + many - 1 of the prefix's and the sequence's own
  const int prefix_blocks = (prefix_rows + 63) >> 6, blocks = prefix_blocks + ((own_rows + 63) >> 6), per = (blocks + parts - 1) / parts;
  const int first = min(blocks, part * per), many = min(blocks - first, per);
  const int skip = min(first, prefix_blocks), own_skip = first - skip, of_prefix = min(many, prefix_blocks - skip);
  w.keys[0] = reinterpret_cast<const uint16_t*>(a.prefix_keys) + at + (size_t)skip * 64 * HD;
  w.values[0] = reinterpret_cast<const uint16_t*>(a.prefix_values) + at + (size_t)skip * 64 * HD;
  w.keys[1] = reinterpret_cast<const uint16_t*>(a.keys) + own + (size_t)own_skip * 64 * HD;
  w.values[1] = reinterpret_cast<const uint16_t*>(a.values) + own + (size_t)own_skip * 64 * HD;
  w.rows[0] = min(prefix_rows - skip * 64, of_prefix * 64);
  w.rows[0] = max(w.rows[0], 0);
  w.rows[1] = max(min(own_rows - own_skip * 64, (many - of_prefix) * 64), 0);
  w.before -= (long long)own_skip * 64;
  RunningRow<HD> row[U];
  meet_many<HD, QT, U>(a, w, row, lds0);
  if (parts > 1) {
    leave_part<HD, U>(a, w, row, part);
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float l = quad_sum(row[u].l);
    const int n = w.first + 16 * (U * wave + u) + r;
    if (n >= w.queries) continue;
    int head;
    const int token = divide(n, a.by_share, head);
    head += hk * share;
    const float inv = token < there && (l > 0.f || l != l) ? 1.0f / l : 0.f;
    const bool zero = inv == 0.f;
    uint16_t* to = a.out + (((size_t)b * a.tokens + token) * a.heads + head) * HD + 4 * g;
#pragma unroll
    for (int t = 0; t < HD / 16; ++t) {
      const f32x4_t o = row[u].o[t];
      *reinterpret_cast<u32x2_t*>(to + 16 * t) =
          zero ? u32x2_t{0u, 0u} : u32x2_t{pack2_bf16(o[0] * inv, o[1] * inv), pack2_bf16(o[2] * inv, o[3] * inv)};
    }
  }
}

// ---- the parts of a query put together: a wave a query, lane p holding part p's (m, sum).  The first kFirst parts' sums are asked for beside them.
__device__ __forceinline__ float wave_max(float v) {
  v = quad_max(v);   // over lanes l, l ^ 16, l ^ 32, l ^ 48
  v = fmaxf(v, row_ror<8>(v));
  v = fmaxf(v, row_ror<4>(v));
  v = fmaxf(v, row_ror<2>(v));
  return fmaxf(v, row_ror<1>(v));
}
template <int HD>
__global__ __launch_bounds__(256) void shared_attention_merge_kernel(SharedAttention a) {
  constexpr int kEach = HD == 128 ? 2 : 1, kLanes = HD / kEach, kFirst = 8;   // components of a lane, lanes that hold some
  const long long place = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (place >= a.queries) return;
  const int lane = threadIdx.x & 63, parts = a.prefix_parts + a.own_parts;
  const float2 ml = a.part_ml[min(lane, parts - 1) * a.queries + place];
  const float* from = a.part_sums + place * HD + kEach * min(lane, kLanes - 1);
  const size_t apart = (size_t)a.queries * HD;
  float x[kFirst][kEach];
  auto ask = [&](int first) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kFirst; ++i) {
      const float* at = from + min(first + i, parts - 1) * apart;
      if constexpr (kEach == 2) {
        const float2 v = *reinterpret_cast<const float2*>(at);
        x[i][0] = v.x;
        x[i][kEach - 1] = v.y;
      } else {
        x[i][0] = *at;
      }
    }
  };
  ask(0);
  int t, h;
  const int b = divide(divide((int)place, a.by_tokens, t), a.by_heads, h);
  const bool there = a.counts == nullptr || t < a.counts[b];
  const float mine = lane < parts && there ? ml.x : -INFINITY;
  const float top = wave_max(mine);
  const float weight = mine == -INFINITY ? 0.f : exp2_hw(mine - top);
  const float l = wave_sum(weight != 0.f ? ml.y * weight : 0.f);
  float o[kEach] = {};
  for (int first = 0; first < parts; first += kFirst) {
    if (first > 0) ask(first);
#pragma unroll
    for (int i = 0; i < kFirst; ++i) {
      // (a lane behind the parts weighs nothing)
      const float c = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), first + i));
#pragma unroll
      for (int e = 0; e < kEach; ++e) o[e] += x[i][e] * c;
    }
  }
  if (lane >= kLanes) return;
  const bool some = l > 0.f || l != l;
  uint16_t* to = a.out + (((size_t)b * a.tokens + t) * a.heads + h) * HD + kEach * lane;
  if constexpr (kEach == 2) *reinterpret_cast<uint32_t*>(to) = some ? pack2_bf16(o[0] / l, o[kEach - 1] / l) : 0u;
  else *to = some ? f32_to_bf16_rne(o[0] / l) : (uint16_t)0;
}

}  // namespace ajq
