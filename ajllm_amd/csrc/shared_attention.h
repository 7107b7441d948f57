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
#include "prefill_attention.h"  // dma16, the fragment reads, pack8_bf16

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
  float scale2;         // log2(e) / sqrt(HD)
};

__device__ __forceinline__ int held(long long n, int most) { return (int)min(max(n, 0ll), (long long)most); }

// What a workgroup works on: a tile of the queries that meet one run of rows.
template <typename CacheT> struct Meeting {
  const CacheT *keys, *values;   // of the (group or sequence, key head)
  int key_head, first_sequence;  // the queries are those of `sequences` sequences from here on and of the key head's heads
  int queries;                   // sequences * tokens * share
  int first;                     // the tile's first query
  int begin, end;                // rows
  bool own;
  long long before;              // own rows a sequence's first new token sees ahead of its own row
};

// query number n of a meeting -> its place in q (and of its partial results), the token
__device__ __forceinline__ long long query_place(const SharedAttention& a, int key_head, int first_sequence, int n, int& token) {
  const int share = a.heads / a.kv_heads, each = a.tokens * share;
  const int sequence = n / each, rest = n - sequence * each;
  token = rest / share;
  const int head = key_head * share + (rest - token * share);
  return ((long long)(first_sequence + sequence) * a.heads + head) * a.tokens + token;
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
__device__ __forceinline__ void load8_halves(const float* p, u32x4_t* to) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  split8(v, to[0], to[1]);
}
__device__ __forceinline__ void load8_halves(const uint16_t* p, u32x4_t* to) { to[0] = *reinterpret_cast<const u32x4_t*>(p); }

// The running softmax of 16 queries, one a lane & 15: m, the lane's own part of the sum, and HD / 16 accumulators of O^T.
template <int HD> struct RunningRow {
  f32x4_t o[HD / 16];
  float m, l;
  bool fresh;   // no visible row met yet
};

// N exponents' products (N 16-key tiles of scores, scaled here) -> probabilities.  The reference point m moves where a lane's sum passes
// kPfTrigger, to the largest exponent where that is past the slack (prefill_attention.h).
template <int HD, int N>
__device__ __forceinline__ void to_probabilities(RunningRow<HD>& row, const f32x4_t (&sc)[N], float scale2, float (&p)[4 * N]) {
  float x[4 * N], sum = 0.f;
#pragma unroll
  for (int e = 0; e < 4 * N; ++e) {
    x[e] = __builtin_fmaf(sc[e >> 2][e & 3], scale2, -row.m);
    p[e] = exp2_hw(x[e]);
    sum += p[e];
  }
  if (__builtin_amdgcn_ballot_w64(row.fresh || sum > kPfTrigger) != 0) {
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < 4 * N; ++e) mx = fmaxf(mx, x[e]);
    mx = quad_max(mx);
    const bool move = row.fresh ? mx > -INFINITY : mx > kPfSlack;
    const float shift = move ? mx : 0.f;
    const float corr = move && !row.fresh ? exp2_hw(-shift) : 1.0f;
    sum = 0.f;
#pragma unroll
    for (int e = 0; e < 4 * N; ++e) {
      p[e] = exp2_hw(x[e] - shift);
      sum += p[e];
    }
    row.m += shift;
    row.l *= corr;
    row.fresh = row.fresh && !move;
#pragma unroll
    for (int t = 0; t < HD / 16; ++t) row.o[t] *= corr;
  }
  row.l += sum;
}

// ---- Few queries: the four waves of a workgroup take blocks of 32 rows in turn, each for itself (no barrier until the end), and RT tiles of 16
// queries meet every row fetched.  What bounds it is memory: a wave asks for the next block's keys as soon as it has used this block's, and for
// its values likewise; eight waves a CU (bf16) then have 64 to 128 KB on their way.
// LDS of a wave: keys, then values, 32 rows each; fp32 rows as two planes of bf16, through registers.
template <int HD, typename CacheT> constexpr int few_wave_bytes() { return 2 * 32 * 2 * HD * kHalves<CacheT>; }
template <int HD, typename CacheT, int RT> constexpr int few_lds_bytes() {
  constexpr int walk = 4 * few_wave_bytes<HD, CacheT>(), join = 4 * RT * 16 * HD * 4;
  return (walk > join ? walk : join) + 4 * RT * 16 * 8;
}

template <int HD, typename QT, typename CacheT, int RT>
__device__ __forceinline__ void meet_few(const SharedAttention& a, const Meeting<CacheT>& w, int part, unsigned char* lds, uint32_t lds0) {
  constexpr int RB = 2 * HD, C = HD / 8, KS = HD / 32, TT = HD / 16, KH = kHalves<CacheT>, QH = kHalves<QT>;
  constexpr int kPlane = 32 * RB;                 // 32 rows of bf16
  constexpr bool kDma = KH == 1;
  constexpr int kRows = 1024 / RB;                // rows of one wave-wide request
  constexpr int kAsk = 32 / kRows;                // requests a block of keys (or values)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t mine = lds0 + (uint32_t)(wave * few_wave_bytes<HD, CacheT>());
  unsigned char* mine_p = lds + wave * few_wave_bytes<HD, CacheT>();

  // ---- queries: fragments of RT tiles, and how many of the meeting's rows each sees
  u32x4_t qf[RT][KS][QH];
  int limit[RT];
#pragma unroll
  for (int u = 0; u < RT; ++u) {
    int token;
    const long long place = query_place(a, w.key_head, w.first_sequence, min(w.first + 16 * u + r, w.queries - 1), token);
    limit[u] = w.own ? held(w.before + token + 1, w.end) : w.end;
#pragma unroll
    for (int s = 0; s < KS; ++s) load8_halves(reinterpret_cast<const QT*>(a.q) + place * HD + 32 * s + 8 * g, qf[u][s]);
  }
  RunningRow<HD> row[RT];
#pragma unroll
  for (int u = 0; u < RT; ++u) {
    row[u].m = row[u].l = 0.f;
    row[u].fresh = true;
#pragma unroll
    for (int t = 0; t < TT; ++t) row[u].o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  // ---- rows on their way (past the last: the last again, which is there and finite)
  const int ask_row = lane / C, slot = lane % C;
  auto ask = [&](const CacheT* from, int at, uint32_t to, bool values) {
    const CacheT* base = from + (size_t)at * HD;
#pragma unroll
    for (int i = 0; i < kAsk; ++i) {
      const int k = kRows * i + ask_row;
      const uint32_t chunk = values ? (uint32_t)((((slot >> 1) ^ (k & (TT - 1))) << 1) | (slot & 1)) : (uint32_t)(slot ^ (k & (C - 1)));
      dma16(base, (uint32_t)(min(k, w.end - 1 - at) * RB) + chunk * 16u, to + (uint32_t)(i * 1024));
    }
  };
  constexpr int kPieces = kDma ? 1 : 32 * C / 64;   // 8 components each, a lane
  Raw8F32 kraw[kPieces], vraw[kPieces];
  auto fetch = [&](int at) {
    if constexpr (!kDma) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int piece = lane + 64 * i, k = min(at + piece / C, w.end - 1);
        kraw[i] = load8_raw(w.keys + (size_t)k * HD + 8 * (piece % C));
        vraw[i] = load8_raw(w.values + (size_t)k * HD + 8 * (piece % C));
      }
    }
  };
  auto lay_down = [&]() {
    if constexpr (!kDma) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int piece = lane + 64 * i, k = piece / C, c = piece % C;
        u32x4_t hi, lo;
        auto put = [&](const Raw8F32& x, unsigned char* to) {
          const float v[8] = {x.a.x, x.a.y, x.a.z, x.a.w, x.b.x, x.b.y, x.b.z, x.b.w};
          split8(v, hi, lo);
          *reinterpret_cast<u32x4_t*>(to) = hi;
          *reinterpret_cast<u32x4_t*>(to + kPlane) = lo;
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

  int at = w.begin + 32 * wave;
  if (at < w.end) {
    if constexpr (kDma) {
      ask(w.keys, at, mine, false);
      ask(w.values, at, values0, true);
    } else {
      fetch(at);
    }
  }
  for (; at < w.end; at += 128) {
    const bool more = at + 128 < w.end;
    if constexpr (kDma) {
      // (behind this block's keys only its values are on their way)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kAsk) : "memory");
    } else {
      lay_down();
      if (more) fetch(at + 128);
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
        ask(w.keys, at + 128, mine, false);
      }
    }
    u32x4_t pf[RT];
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      if (__builtin_amdgcn_ballot_w64(at + 32 > limit[u]) != 0) {
#pragma unroll
        for (int jb = 0; jb < 2; ++jb)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (at + 16 * jb + 4 * g + i >= limit[u]) sc[u][jb][i] = -INFINITY;
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
        ask(w.values, at + 128, values0, true);
      }
    } else {
      wave_lds_order();
    }
  }

  // ---- the four waves' results meet in LDS
  __syncthreads();
  constexpr int kJoin = RT * 16;   // queries
  float* sums = reinterpret_cast<float*>(lds);
  float2* ml = reinterpret_cast<float2*>(lds + few_lds_bytes<HD, CacheT, RT>() - 4 * RT * 16 * 8);
#pragma unroll
  for (int u = 0; u < RT; ++u) {
    const float l = quad_sum(row[u].l);
    if (g == 0) ml[wave * kJoin + 16 * u + r] = float2{row[u].fresh && l == 0.f ? -INFINITY : row[u].m, l};   // (NaN stays)
#pragma unroll
    for (int t = 0; t < TT; ++t)
      *reinterpret_cast<f32x4_t*>(sums + ((size_t)(wave * kJoin + 16 * u + r)) * HD + 16 * t + 4 * g) = row[u].o[t];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kJoin * (HD / 4); i += 256) {
    const int n = i / (HD / 4), d = 4 * (i % (HD / 4));
    if (w.first + n >= w.queries) break;   // (n only grows)
    float2 e[4];
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      e[k] = ml[k * kJoin + n];
      m = fmaxf(m, e[k].x);
    }
    float l = 0.f;
    f32x4_t o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float weight = e[k].x == -INFINITY ? 0.f : exp2_hw(e[k].x - m);
      l += e[k].y * weight;
      o += *reinterpret_cast<const f32x4_t*>(sums + (size_t)(k * kJoin + n) * HD + d) * weight;
    }
    int token;
    const long long place = query_place(a, w.key_head, w.first_sequence, w.first + n, token) + part * a.queries;
    if (d == 0) a.part_ml[place] = float2{m, l};
    *reinterpret_cast<f32x4_t*>(a.part_sums + place * HD + d) = o;
  }
}

// ---- Many queries on bf16 rows: 128 to a workgroup, 32 to each wave, all four walking the same blocks of 64 rows (LDS, two stages, one barrier a
// block, as attn_prefill_kernel).  Bound by MFMA.  The walk goes over a run of the group's prefix and, behind it, of one sequence's own
// rows; either may be empty.
template <typename CacheT> struct Walk {
  const CacheT *keys[2], *values[2];   // prefix, own
  int rows[2];                         // of which so many are there
  int first_block, blocks;             // the walk's part of the blocks of both
  int key_head, first_sequence, queries, first;
  long long before;
};
template <int HD> constexpr int many_lds_bytes() { return 4 * 64 * 2 * HD; }

template <int HD, typename QT>
__device__ __forceinline__ void meet_many(const SharedAttention& a, const Walk<uint16_t>& w, RunningRow<HD> (&row)[2], uint32_t lds0) {
  constexpr int RB = 2 * HD, C = HD / 8, KS = HD / 32, TT = HD / 16, QH = kHalves<QT>;
  constexpr int kTile = 64 * RB;
  constexpr int kReqRows = 1024 / RB;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int prefix_blocks = (w.rows[0] + 63) >> 6;

  const int krow = kReqRows * wave + lane / C, slot = lane % C;
  const uint32_t k_chunk = (uint32_t)(slot ^ (krow & (C - 1)));
  const uint32_t v_chunk = (uint32_t)((((slot >> 1) ^ (krow & (TT - 1))) << 1) | (slot & 1));
  // part i (of KS) of block j: this wave's kReqRows rows of the i-th group of 4 kReqRows
  auto ask = [&](int j, int i) {
    const int own = w.first_block + j >= prefix_blocks, kb0 = (w.first_block + j - (own ? prefix_blocks : 0)) * 64;
    const uint32_t to = lds0 + (uint32_t)((j & 1) * 2 * kTile + (wave + 4 * i) * 1024);
    const uint32_t at = (uint32_t)(min(4 * kReqRows * i + krow, w.rows[own] - 1 - kb0) * RB);
    dma16(w.keys[own] + (size_t)kb0 * HD, at + k_chunk * 16u, to);
    dma16(w.values[own] + (size_t)kb0 * HD, at + v_chunk * 16u, to + (uint32_t)kTile);
  };
  uint32_t k_rd[KS], v_rd[TT];
#pragma unroll
  for (int s = 0; s < KS; ++s) k_rd[s] = lds0 + (uint32_t)(r * RB + 16 * ((4 * s + g) ^ (r & (C - 1))));
  const int vkey = 4 * g + (r >> 2);
#pragma unroll
  for (int t = 0; t < TT; ++t) v_rd[t] = lds0 + (uint32_t)(kTile + vkey * RB + 32 * (t ^ (vkey & (TT - 1))) + 8 * (r & 3));

#pragma unroll
  for (int i = 0; i < KS; ++i) ask(0, i);
  u32x4_t qf[2][KS][QH];
  int limit[2], nearest, farthest;   // own rows that a lane's queries see, that the wave's first and last one see
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    int token;
    const long long place = query_place(a, w.key_head, w.first_sequence, min(w.first + 32 * wave + 16 * u + r, w.queries - 1), token);
    limit[u] = held(w.before + token + 1, w.rows[1]);
#pragma unroll
    for (int s = 0; s < KS; ++s) load8_halves(reinterpret_cast<const QT*>(a.q) + place * HD + 32 * s + 8 * g, qf[u][s]);
    row[u].m = row[u].l = 0.f;
    row[u].fresh = true;
#pragma unroll
    for (int t = 0; t < TT; ++t) row[u].o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  nearest = __builtin_amdgcn_readlane(limit[0], 0);
  farthest = __builtin_amdgcn_readlane(limit[1], 63);
  const bool idle = w.first + 32 * wave >= w.queries;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  for (int j = 0; j < w.blocks; ++j) {
    const bool own = w.first_block + j >= prefix_blocks;
    const int kb0 = (w.first_block + j - (own ? prefix_blocks : 0)) * 64;
    const bool more = j + 1 < w.blocks;
    if (idle || (own && kb0 >= farthest)) {
      if (more) {
#pragma unroll
        for (int i = 0; i < KS; ++i) ask(j + 1, i);
      }
    } else {
      f32x4_t sc[2][4];
      u32x4_t ka[4];
#pragma unroll
      for (int jb = 0; jb < 4; ++jb) ka[jb] = pf_read128(k_rd[0] + (uint32_t)(jb * 16 * RB));
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        u32x4_t kn[4];
        if (s < KS - 1) {
#pragma unroll
          for (int jb = 0; jb < 4; ++jb) kn[jb] = pf_read128(k_rd[s + 1] + (uint32_t)(jb * 16 * RB));
        }
#pragma unroll
        for (int qh = 0; qh < QH; ++qh)
#pragma unroll
          for (int jb = 0; jb < 4; ++jb)
#pragma unroll
            for (int u = 0; u < 2; ++u) sc[u][jb] = mfma16(ka[jb], qf[u][s][qh], s + qh == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : sc[u][jb]);
        if (more) ask(j + 1, s);
        if (s < KS - 1) {
#pragma unroll
          for (int jb = 0; jb < 4; ++jb) ka[jb] = kn[jb];
        }
      }
      const int seen = own ? nearest : w.rows[0];
      if (kb0 + 64 > seen) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int last = own ? limit[u] : w.rows[0];
#pragma unroll
          for (int jb = 0; jb < 4; ++jb)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (kb0 + 16 * jb + 4 * g + i >= last) sc[u][jb][i] = -INFINITY;
        }
      }
      u32x4_t pf[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float p[16];
        to_probabilities<HD, 4>(row[u], sc[u], a.scale2, p);
        pf[u][0] = pack8_bf16(&p[0]);
        pf[u][1] = pack8_bf16(&p[8]);
      }
      constexpr int kRing = TT < 8 ? TT : 8;
      auto v_lo = [&](int i) { return pf_read_tr(v_rd[i % TT] + (uint32_t)((i / TT) * 32 * RB)); };
      auto v_hi = [&](int i) { return pf_read_tr(v_rd[i % TT] + (uint32_t)((i / TT) * 32 * RB + 16 * RB)); };
      u32x2_t vlo[kRing], vhi[kRing];
#pragma unroll
      for (int i = 0; i < kRing; ++i) {
        vlo[i] = v_lo(i);
        vhi[i] = v_hi(i);
      }
#pragma unroll
      for (int i = 0; i < 2 * TT; ++i) {
        const u32x4_t vf = {vlo[i % kRing].x, vlo[i % kRing].y, vhi[i % kRing].x, vhi[i % kRing].y};
#pragma unroll
        for (int u = 0; u < 2; ++u) row[u].o[i % TT] = mfma16(vf, pf[u][i / TT], row[u].o[i % TT]);
        if (i + kRing < 2 * TT) {
          vlo[i % kRing] = v_lo(i + kRing);
          vhi[i % kRing] = v_hi(i + kRing);
        }
      }
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) k_rd[s] ^= (uint32_t)(2 * kTile);
#pragma unroll
    for (int t = 0; t < TT; ++t) v_rd[t] ^= (uint32_t)(2 * kTile);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }
}

// a lane's queries of meet_many as partial results
template <int HD>
__device__ __forceinline__ void leave_part(const SharedAttention& a, const Walk<uint16_t>& w, const RunningRow<HD> (&row)[2], int part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const float l = quad_sum(row[u].l);
    const int n = w.first + 32 * wave + 16 * u + r;
    if (n >= w.queries) continue;
    int token;
    const long long place = query_place(a, w.key_head, w.first_sequence, n, token) + part * a.queries;
    if (g == 0) a.part_ml[place] = float2{row[u].fresh && l == 0.f ? -INFINITY : row[u].m, l};
#pragma unroll
    for (int t = 0; t < HD / 16; ++t) *reinterpret_cast<f32x4_t*>(a.part_sums + place * HD + 16 * t + 4 * g) = row[u].o[t];
  }
}

// A launch's workgroups: first the prefix's (a part of a (group, key head)'s rows and a tile of queries each; those that share rows are next
// to each other on one XCD), then the sequences' own likewise.
template <typename CacheT, int HD>
__device__ __forceinline__ bool find_meeting(const SharedAttention& a, int tile_queries_prefix, int tile_queries_own, Meeting<CacheT>& w, int& part) {
  const int share = a.heads / a.kv_heads;
  w.own = (int)blockIdx.x >= a.prefix_blocks;
  const int id = (int)blockIdx.x - (w.own ? a.prefix_blocks : 0);
  const int tiles = w.own ? a.own_tiles : a.prefix_tiles, parts = w.own ? a.own_parts : a.prefix_parts;
  const int runs = (w.own ? a.batch : a.groups) * a.kv_heads * parts;      // of rows
  const int run = (id & 7) + 8 * (id / (8 * tiles)), tile = (id >> 3) % tiles;
  if (run >= runs) return false;
  part = run % parts;
  const int unit = run / parts;
  w.key_head = unit % a.kv_heads;
  const int outer = unit / a.kv_heads, each = a.batch / a.groups;
  const long long off = a.offset ? *a.offset : 0ll;
  int there = a.tokens, rows;
  if (w.own) {
    w.first_sequence = outer;
    w.queries = a.tokens * share;
    w.before = a.rows[outer] + off;
    if (a.counts) there = held(a.counts[outer], a.tokens);
    rows = held(w.before + there, a.max_len);
    const size_t at = (size_t)outer * a.cache_batch + (size_t)w.key_head * a.cache_head;
    w.keys = reinterpret_cast<const CacheT*>(a.keys) + at;
    w.values = reinterpret_cast<const CacheT*>(a.values) + at;
  } else {
    w.first_sequence = outer * each;
    w.queries = each * a.tokens * share;
    w.before = 0;
    rows = held(a.prefix_lengths[outer], a.prefix_cap);
    const size_t at = (size_t)outer * a.prefix_group + (size_t)w.key_head * a.prefix_head;
    w.keys = reinterpret_cast<const CacheT*>(a.prefix_keys) + at;
    w.values = reinterpret_cast<const CacheT*>(a.prefix_values) + at;
  }
  w.first = tile * (w.own ? tile_queries_own : tile_queries_prefix);
  // parts of whole blocks of 32 rows
  const int per = ((rows + parts - 1) / parts + 31) & ~31;
  w.begin = (int)min((long long)rows, (long long)part * per);
  w.end = min(rows, w.begin + per);
  if (w.own) part += a.prefix_parts;
  return true;
}

template <int HD, typename QT, typename CacheT, int RTP, int RTO>
__global__ __launch_bounds__(256, sizeof(CacheT) == 4 ? 1 : 2) void shared_attention_few_kernel(SharedAttention a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char shared_lds[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(pf_lds_char_t*)shared_lds;
  Meeting<CacheT> w;
  int part;
  if (!find_meeting<CacheT, HD>(a, 16 * RTP, 16 * RTO, w, part)) return;
  if (RTP == RTO || !w.own) meet_few<HD, QT, CacheT, RTP>(a, w, part, shared_lds, lds0);
  else meet_few<HD, QT, CacheT, RTO>(a, w, part, shared_lds, lds0);
}

// The prefix by meet_many, the sequences' own rows by meet_few.
template <int HD, typename QT, int RTO>
__global__ __launch_bounds__(256, 2) void shared_attention_many_kernel(SharedAttention a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char shared_lds[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(pf_lds_char_t*)shared_lds;
  Meeting<uint16_t> w;
  int part;
  if (!find_meeting<uint16_t, HD>(a, 128, 16 * RTO, w, part)) return;
  if (w.own) {
    meet_few<HD, QT, uint16_t, RTO>(a, w, part, shared_lds, lds0);
    return;
  }
  Walk<uint16_t> walk;
  walk.keys[0] = w.keys + (size_t)w.begin * HD;
  walk.values[0] = w.values + (size_t)w.begin * HD;
  walk.keys[1] = walk.values[1] = nullptr;
  walk.rows[0] = w.end - w.begin;
  walk.rows[1] = 0;
  walk.first_block = 0;
  walk.blocks = (walk.rows[0] + 63) >> 6;
  walk.key_head = w.key_head;
  walk.first_sequence = w.first_sequence;
  walk.queries = w.queries;
  walk.first = w.first;
  walk.before = 0;
  RunningRow<HD> row[2];
  if (walk.blocks > 0) {
    meet_many<HD, QT>(a, walk, row, lds0);
  } else {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      row[u].m = row[u].l = 0.f;
      row[u].fresh = true;
#pragma unroll
      for (int t = 0; t < HD / 16; ++t) row[u].o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  }
  leave_part<HD>(a, walk, row, part);
}

// Sequences with many new tokens each: 128 queries of one sequence walk the prefix and then its own rows, and what comes out is the result.  With
// own_parts > 1 the walk is cut up and leaves parts for the merge.
template <int HD, typename QT>
__global__ __launch_bounds__(256, 2) void shared_attention_walk_kernel(SharedAttention a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char shared_lds[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(pf_lds_char_t*)shared_lds;
  const int share = a.heads / a.kv_heads, parts = a.own_parts, tiles = a.own_tiles;
  const int id = (int)blockIdx.x, run = (id & 7) + 8 * (id / (8 * tiles * parts)), rest = (id >> 3) % (tiles * parts);
  if (run >= a.batch * a.kv_heads) return;
  const int tile = tiles - 1 - rest / parts, part = rest % parts;
  const int b = run / a.kv_heads, hk = run % a.kv_heads, group = b / (a.batch / a.groups);
  Walk<uint16_t> w;
  w.key_head = hk;
  w.first_sequence = b;
  w.queries = a.tokens * share;
  w.first = 128 * tile;
  w.before = a.rows[b] + (a.offset ? *a.offset : 0ll);
  const int there = a.counts ? held(a.counts[b], a.tokens) : a.tokens;
  const int last = min((w.first + 127) / share, there - 1);          // the tile's last token that is there
  const size_t at = (size_t)group * a.prefix_group + (size_t)hk * a.prefix_head, own = (size_t)b * a.cache_batch + (size_t)hk * a.cache_head;
  w.keys[0] = reinterpret_cast<const uint16_t*>(a.prefix_keys) + at;
  w.values[0] = reinterpret_cast<const uint16_t*>(a.prefix_values) + at;
  w.keys[1] = reinterpret_cast<const uint16_t*>(a.keys) + own;
  w.values[1] = reinterpret_cast<const uint16_t*>(a.values) + own;
  const bool none = w.first >= there * share;
  w.rows[0] = none ? 0 : held(a.prefix_lengths[group], a.prefix_cap);
  w.rows[1] = none ? 0 : held(w.before + last + 1, a.max_len);
  const int blocks = ((w.rows[0] + 63) >> 6) + ((w.rows[1] + 63) >> 6), per = (blocks + parts - 1) / parts;
  w.first_block = min(blocks, part * per);
  w.blocks = min(blocks - w.first_block, per);
  RunningRow<HD> row[2];
  if (w.blocks > 0) {
    meet_many<HD, QT>(a, w, row, lds0);
  } else {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      row[u].m = row[u].l = 0.f;
      row[u].fresh = true;
#pragma unroll
      for (int t = 0; t < HD / 16; ++t) row[u].o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  }
  if (parts > 1) {
    leave_part<HD>(a, w, row, part);
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const float l = quad_sum(row[u].l);
    const int n = w.first + 32 * wave + 16 * u + r;
    if (n >= w.queries) continue;
    const int token = n / share, head = hk * share + (n - token * share);
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

// ---- the parts of a query put together: a wave a query, lane p holding part p's (m, sum)
template <int HD>
__global__ __launch_bounds__(256) void shared_attention_merge_kernel(SharedAttention a) {
  const long long place = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (place >= a.queries) return;
  const int lane = threadIdx.x & 63, parts = a.prefix_parts + a.own_parts;
  const int t = (int)(place % a.tokens), h = (int)(place / a.tokens % a.heads), b = (int)(place / a.tokens / a.heads);
  const float2 ml = a.part_ml[min(lane, parts - 1) * a.queries + place];
  constexpr int kLanes = HD / 2;                   // that hold two components
  const int dl = min(lane, kLanes - 1);
  const bool there = a.counts == nullptr || t < a.counts[b];
  const float mine = lane < parts && there ? ml.x : -INFINITY;
  float top = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off));
  const float weight = mine == -INFINITY ? 0.f : exp2_hw(mine - top);
  const float l = wave_sum(lane < parts && weight != 0.f ? ml.y * weight : 0.f);
  float2 o = float2{0.f, 0.f};
#pragma unroll 8
  for (int p = 0; p < parts; ++p) {
    const float c = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), p));
    const float2 x = *reinterpret_cast<const float2*>(a.part_sums + (p * a.queries + place) * HD + 2 * dl);
    o.x += x.x * c;
    o.y += x.y * c;
  }
  if (lane >= kLanes) return;
  const uint32_t to = l > 0.f || l != l ? pack2_bf16(o.x / l, o.y / l) : 0u;
  reinterpret_cast<uint32_t*>(a.out + (((size_t)b * a.tokens + t) * a.heads + h) * HD)[lane] = to;
}

}  // namespace ajq
