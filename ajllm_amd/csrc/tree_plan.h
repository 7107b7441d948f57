// How a call of tree attention is cut up and which way it goes: host arithmetic alone, by what the host knows.
#pragma once
#include <math.h>
#include <stddef.h>

#include <algorithm>

#include "../../include/ajq_draft.h"
#include "../../include/ajq_serve.h"   // element types
#include "host_math.h"

namespace ajq {
constexpr int kMostDealt = 64;   // sequences that parts are dealt out to: a lane each
}

namespace {

using ajq::kMostDealt;

// How a call is cut up: tiles of a sequence's queries of a key head, parts of its rows.  The lengths are on the device: max_len is what they can be.
struct TreePlan {
  bool walk;     // tiles of 16 rt queries a wave, by meet_many or (fp32 caches) tree_attention_laid_kernel; else of 16 rt, by meet_few
  int rt, waves, tiles;
  bool alone;    // a wave has a tile and its rows to itself
  int runs;      // 0: every sequence's rows are one part
  long long blocks, queries;
  size_t bytes;
};
constexpr int kMostParts = 64;      // of a sequence: a lane each in the merge

// What a call takes, in us, from what bounds it:
//   a launch, and a wave's own part of it;   the steps of its longest workgroup, each of which takes the longer the more waves share a SIMD, for every round of
//   workgroups;   the rows from memory, and again from L2 for every other tile;   a second launch that puts the parts together, and their way through memory.
// The constants fit 6059 calls (1 to 24 sequences, 1 to 128 tokens, five layouts of heads, 60 to 24000 rows) to 11 to 14 %; what is chosen by them takes 2 to 3 % longer
// (geometric mean) than the fastest of what was tried.  Where the ways part, for instance (us; heads / key heads x size, tokens, rows): 32 / 8 x 128, 1 x 8 behind 500: tiles of 16
// in one launch 6.3, of 32 9.1, in seven parts 7.2; 6 x 32 behind 2000: tiles of 32 and eight waves in one launch 18.5, four waves in 16 runs 22.0; 6 x 32 behind 12000: in 16
// runs 56.7, eight waves in one launch 2.2 times that; 8 x 64 behind 32768: tiles of 256 of eight waves in 28 runs 254, of 128 of four 324.
// fp32 rows laid down once: 1881 calls to 10 %; what is chosen with them takes 4 % longer than the fastest of 350 calls' ways.  Rows and tokens of all these calls, and of the
// examples, are the largest of the batch: the others have from a half of that on.
struct TreeCost {
  float start, per_waves, per_tiles, step, step_dim, step_tiles, crowd, memory, merge, merge_bytes, l2;
};
constexpr TreeCost kFewBf16{3.854f, 0.596f, 1.229f, 0.249f, 0.54f, 0.36f, 0.319f, 6.172f, 2.349f, 0.709f, 47.1f};
constexpr TreeCost kWalkBf16{6.769f, 1.665f, 2.713f, 0.295f, 0.418f, 0.215f, 0.433f, 5.035f, 2.249f, 0.404f, 18.64f};
constexpr TreeCost kLaidF32{4.405f, 0.f, 1.314f, 0.29f, 0.948f, 0.563f, 0.222f, 6.547f, 2.973f, 0.619f, 46.78f};
constexpr TreeCost kFewF32{3.243f, 0.f, 1.392f, 0.156f, 3.167f, 0.f, 0.63f, 5.781f, 3.079f, 0.922f, 39.38f};
float tree_cost(const ajqt_tree_attention_args* a, const TreePlan& p) {
  const bool bf16 = a->cache_dtype == AJQS_BF16;
  const TreeCost& c = p.walk ? (bf16 ? kWalkBf16 : kLaidF32) : bf16 ? kFewBf16 : kFewF32;
  const float dim = (float)a->dim / 128.f, batch = (float)a->batch, waves = (float)p.waves, kv = (float)a->kv_heads;
  // rows: of the longest sequence the whole capacity (one run is one workgroup's), of several three quarters on average, as if lengths lay between a half of it and all.  What is
  // filled is not known here: a cache of 32784 rows that holds 272 is read in 32 runs, 14.2 us instead of 5.8 (8 x 16, 32 / 8 x 128, bf16).
  const float longest = (float)a->max_len, mean = a->batch == 1 ? longest : 0.75f * longest;
  const float rows = !p.runs ? longest : a->batch == 1 ? longest / (float)p.runs : batch * mean / ((float)p.runs - 0.5f * batch);
  const float steps = ceilf(!p.walk ? rows / (32.f * waves) : bf16 ? rows / 64.f : rows / 32.f);
  const float workgroups = (p.runs ? (float)p.runs : batch) * kv * (float)p.tiles;
  const float at_once = (!bf16 && !p.walk && p.rt == 2 ? 4.f : 8.f) / dim;   // waves a CU, by registers and LDS
  const float rounds = fmaxf(1.f, workgroups * waves / (256.f * at_once)), crowd = fmaxf(1.f, fminf(ceilf(workgroups / 256.f) * waves, at_once) / 4.f);
  const float work = rounds * steps * (c.step + (c.step_dim + c.step_tiles * (float)(p.rt - 1)) * dim) * (1.f + c.crowd * (crowd - 1.f));
  const float megabytes = batch * kv * mean * 2.f * (float)a->dim * (bf16 ? 2e-6f : 4e-6f);
  const float memory = megabytes / c.memory + megabytes * (float)(p.tiles - 1) / c.l2;
  const float parts = (float)p.runs * kv * (float)a->tokens * (float)(a->heads / a->kv_heads) * (float)a->dim * 4e-6f;
  return c.start + c.per_waves * (waves / 4.f - 1.f) + c.per_tiles * (float)(p.rt - 1) + cbrtf(work * work * work + memory * memory * memory) +
         (p.runs ? c.merge + c.merge_bytes * parts : 0.f);
}
TreePlan plan_tree(const ajqt_tree_attention_args* a) {
  const long long mine = (long long)a->tokens * (a->heads / a->kv_heads), units = (long long)a->batch * a->kv_heads;
  const bool bf16 = a->cache_dtype == AJQS_BF16;
  TreePlan best{};
  float least = INFINITY;
  for (int walk = 0; walk <= (mine > (bf16 ? 64 : 16)); ++walk) {
    if (!walk && bf16 && mine > 256) continue;
    for (int rt = 1; rt <= 2; ++rt) {
      // (what is not built, or has nothing to do)
      if (!walk ? rt == 2 && mine <= 16 : rt == 2 && (bf16 ? a->q_dtype != AJQS_BF16 || a->dim != 128 : mine <= 64)) continue;
      for (int waves = 4; waves <= 8; waves += 4) {
        if (waves == 8 && (walk ? !bf16 || a->dim < 64 || mine <= 64 * rt : !bf16 && rt == 2 && a->dim == 128)) continue;
        TreePlan p{};
        p.walk = walk != 0;
        p.rt = rt;
        p.waves = waves;
        p.tiles = (int)ceil_div(mine, 16ll * rt * (walk ? waves : 1));
        const long long round = 2048 / waves / (a->kv_heads * (long long)p.tiles);
        const long long most = a->batch * std::min(ceil_div(a->max_len, walk ? 128 : 64), (long long)kMostParts);
        for (int n = 0; n < 4; ++n) {
          p.runs = (int)std::min(most, n == 0 ? 0 : n == 1 ? round / 2 : n == 2 ? round : 2 * round);
          if (n && (p.runs <= a->batch || a->batch > kMostDealt)) continue;
          if (n && !bf16 && !walk && rt == 2 && waves == 4) continue;   // (parts of fp32 rows for so many queries: laid down once they take less, or eight waves do)
          const float cost = tree_cost(a, p);
          if (cost < least) {
            least = cost;
            best = p;
          }
        }
      }
    }
  }
  // Many tiles and few rows: with a wave for each, nothing is put together.  (500 calls of 8 to 64 sequences behind 2 to 400 rows: within these limits 18 % less than by four
  // waves a tile on bf16 rows, 6 % on fp32 ones, none slower by more than 5 %; 45 x 32 heads of 128 behind 5 fp32 rows 6.7 us instead of 12.5, 48 x 24 tokens x 16 behind 84
  // bf16 ones 10.4 instead of 14.5.  Beyond them: 64 x 12 of 64 behind 300 11.3 instead of 10.9, 45 x 32 behind 200 fp32 ones 60 instead of 48.)
  if (!best.walk && units * ceil_div(mine, 16) >= 512 && a->max_len <= (bf16 ? 128 : 64)) {
    best = TreePlan{};
    best.alone = true;
    best.rt = 1;
    best.waves = 4;
    best.tiles = (int)ceil_div(mine, 16);
  }
  best.queries = (long long)a->batch * a->heads * a->tokens;
  best.blocks = best.alone ? ceil_div(units * best.tiles, 4) : ceil_div(best.runs ? (long long)best.runs * a->kv_heads : units, 8) * 8 * best.tiles;
  best.bytes = best.runs ? (size_t)best.runs * a->kv_heads * mine * (8 + 4 * (size_t)a->dim) + 8 * (size_t)a->batch : 0;
  return best;
}

}  // namespace
