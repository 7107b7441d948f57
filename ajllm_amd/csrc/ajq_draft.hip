// C ABI of libajq_draft.so (include/ajq_draft.h): argument validation, launch geometry, error reporting.
#include "serve_host.h"

#include "../../include/ajq_draft.h"
#include "draft_kernels.h"
#include "log_probs_kernels.h"
#include "tree_attention.h"

namespace {

constexpr int kMostRows = 1 << 30;   // of a cache head

int check_tree(const ajqt_tree_attention_args* a) {
  const char* what = "ajqt_tree_attention";
  if (!a) return fail(AJQ_ERR_NULL, "%s: null arguments", what);
  if (!a->q || !a->keys || !a->values || !a->masks || !a->rows || !a->out) return fail(AJQ_ERR_NULL, "%s: null pointer argument", what);
  if (!built_dim(a->dim)) return fail(AJQ_ERR_UNSUPPORTED, "%s: head size %d (128, 64 and 32 are built)", what, a->dim);
  if (a->batch < 1 || a->tokens < 1 || a->kv_heads < 1 || a->heads < 1 || a->heads % a->kv_heads != 0 || a->max_len < 1 || a->max_len > kMostRows ||
      a->tokens > kMostRows)
    return fail(AJQ_ERR_SHAPE, "%s: unsupported shape (batch=%d tokens=%d heads=%d kv_heads=%d max_len=%d)", what, a->batch, a->tokens, a->heads,
                a->kv_heads, a->max_len);
  if ((long long)a->batch * a->heads * a->tokens > 0x1FFFFFFFLL)
    return fail(AJQ_ERR_SHAPE, "%s: too many queries (%d x %d x %d)", what, a->batch, a->heads, a->tokens);
  if (!known(a->q_dtype) || !known(a->cache_dtype)) return fail(AJQ_ERR_UNSUPPORTED, "%s: unknown element type", what);
  if (a->mask_batch < 0 || a->mask_token < 0) return fail(AJQ_ERR_SHAPE, "%s: negative mask stride", what);
  if (!aligned16(a->q) || !aligned16(a->out)) return fail(AJQ_ERR_ALIGN, "%s: q and out must be 16-byte aligned", what);
  if (!aligned4(a->masks)) return fail(AJQ_ERR_ALIGN, "%s: masks must be aligned to their words", what);
  return check_caches(what, a->keys, a->values, a->cache_batch, a->cache_head);
}

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
// fp32 rows laid down once: 1881 calls to 10 %; what is chosen with them takes 4 % longer than the fastest of 350 calls' ways.
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
  // rows: of the longest sequence all (one run is one workgroup's), of several three quarters on average
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

// (A step asks for the same plan a layer, and twice a call: the thread's last one is kept, by what it was made from.)
TreePlan tree_plan(const ajqt_tree_attention_args* a) {
  const int of[] = {a->batch, a->tokens, a->heads, a->kv_heads, a->dim, a->max_len, a->q_dtype, a->cache_dtype};
  static thread_local int last_of[8] = {};
  static thread_local TreePlan last;
  if (!std::equal(of, of + 8, last_of)) {
    last = plan_tree(a);
    std::copy(of, of + 8, last_of);
  }
  return last;
}

TreeAttention tree_of(const ajqt_tree_attention_args* a, const TreePlan& p, void* workspace) {
  TreeAttention s{};
  s.q = a->q;
  s.prefix_keys = s.keys = a->keys;
  s.prefix_values = s.values = a->values;
  s.rows = int64s(a->rows);
  s.counts = int64s(a->counts);
  s.offset = int64s(a->offset);
  s.out = reinterpret_cast<uint16_t*>(a->out);
  s.part_sums = reinterpret_cast<float*>(workspace);
  const size_t partial = (size_t)p.runs * a->kv_heads * a->tokens * (a->heads / a->kv_heads);
  s.part_ml = reinterpret_cast<float2*>(s.part_sums + partial * a->dim);
  s.dealt = reinterpret_cast<int2*>(s.part_ml + partial);
  s.runs = p.runs;
  s.prefix_group = s.cache_batch = a->cache_batch;
  s.prefix_head = s.cache_head = a->cache_head;
  s.queries = p.queries;
  s.groups = s.batch = a->batch;
  s.tokens = a->tokens;
  s.heads = a->heads;
  s.kv_heads = a->kv_heads;
  s.prefix_cap = s.max_len = a->max_len;
  s.own_parts = 1;
  s.own_alone = p.alone;
  s.own_tiles = p.tiles;
  s.scale2 = kLog2e / sqrtf((float)a->dim);
  s.by_share = divide_by(a->heads / a->kv_heads);
  s.by_each = divide_by((long long)a->tokens * (a->heads / a->kv_heads));
  s.by_tokens = divide_by(a->tokens);
  s.by_heads = divide_by(a->heads);
  s.by_kv_heads = divide_by(a->kv_heads);
  s.by_group = divide_by(1);
  s.by_prefix_tiles = s.by_prefix_parts = divide_by(1);
  s.by_own_tiles = divide_by(p.tiles);
  s.by_own_parts = divide_by(1);
  s.masks = a->masks;
  s.mask_batch = a->mask_batch;
  s.mask_token = a->mask_token;
  return s;
}

// Whether the blocks of `size` bytes at the sums of the dimensions' multiples lie apart, one dimension inside the other (any other order is taken to meet).
struct Dimension {
  long long count, stride;   // (bytes)
};
template <size_t N>
bool nested(Dimension (&dims)[N], long long size) {
  std::sort(dims, dims + N, [](const Dimension& x, const Dimension& y) { return x.stride < y.stride; });
  for (const Dimension& d : dims) {
    if (d.count == 1) continue;
    if (d.stride < size) return false;
    size += (d.count - 1) * d.stride;
  }
  return true;
}

int check_log_probs(const ajqt_log_probs_args* a) {
  const char* what = "ajqt_log_probs";
  if (!a) return fail(AJQ_ERR_NULL, "%s: null arguments", what);
  if (!a->logits || !a->entropy || (a->targets && (!a->log_probs || !a->ranks)) || (a->top && (!a->top_log_probs || !a->top_ids)))
    return fail(AJQ_ERR_NULL, "%s: null pointer argument", what);
  if (!known(a->dtype)) return fail(AJQ_ERR_UNSUPPORTED, "%s: unknown element type", what);
  if (a->rows < 1 || a->vocab < 1 || a->ld < 0 || a->top < 0 || a->top > kMostTop || a->top > a->vocab)
    return fail(AJQ_ERR_SHAPE, "%s: unsupported shape (rows=%d vocab=%d ld=%lld top=%d)", what, a->rows, a->vocab, (long long)a->ld, a->top);
  if (!aligned4(a->log_probs) || !aligned4(a->entropy) || !aligned4(a->top_log_probs) || (a->dtype == AJQS_F32 && !aligned4(a->logits)) ||
      (reinterpret_cast<uintptr_t>(a->logits) & 1u))
    return fail(AJQ_ERR_ALIGN, "%s: logits and results must be aligned to their elements", what);
  if (a->rows > kMostLanes / 256) return fail(AJQ_ERR_SHAPE, "%s: %d rows in a launch", what, a->rows);
  return AJQ_OK;
}

// How rows are cut up: slices of about one size, at most what a workgroup's registers hold.
struct LogProbsPlan {
  int lanes, slice;
  long long slices;
  size_t bytes;
};
LogProbsPlan log_probs_plan(const ajqt_log_probs_args* a) {
  LogProbsPlan p{};
  const long long size = a->dtype == AJQS_BF16 ? 2 : 4, piece = 16 / size;
  // (rows that do not begin on 16 bytes fill up the piece they begin in)
  const bool even = aligned16(a->logits) && (a->rows == 1 || a->ld * size % 16 == 0);
  auto most = [&](long long lanes) { return lanes * kLogPieces * piece - (even ? 0 : piece); };
  p.lanes = a->vocab <= most(256) || (a->vocab > most(1024) && a->rows * ceil_div(a->vocab, most(1024)) < 256) ? 256 : 1024;
  p.slices = ceil_div(a->vocab, most(p.lanes));
  p.slice = (int)std::min((long long)a->vocab, std::min(ceil_div(ceil_div(a->vocab, p.slices), 64) * 64, most(p.lanes)));
  p.slices = ceil_div(a->vocab, p.slice);
  p.bytes = p.slices > 1 ? (size_t)a->rows * p.slices * (sizeof(f32x4_t) + 8 * (size_t)a->top) + 4 * (size_t)a->rows : 0;
  return p;
}

}  // namespace

extern "C" {

const char* ajqt_last_error(void) { return g_error; }

size_t ajqt_tree_attention_workspace(const ajqt_tree_attention_args* a) { return check_tree(a) ? 0 : tree_plan(a).bytes; }

int ajqt_tree_attention(const ajqt_tree_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "ajqt_tree_attention";
  if (int e = check_tree(a)) return e;
  const TreePlan p = tree_plan(a);
  if (p.blocks > kMostLanes / (64 * p.waves)) return fail(AJQ_ERR_SHAPE, "%s: too many tiles of queries", what);
  if (p.bytes && ceil_div(p.queries, 4) > kMostLanes / 256) return fail(AJQ_ERR_SHAPE, "%s: too many queries (%lld)", what, p.queries);
  if (p.bytes && (!workspace || workspace_bytes < p.bytes))
    return fail(AJQ_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, p.bytes, workspace_bytes);
  if (!aligned16(workspace)) return fail(AJQ_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", what);
  const TreeAttention s = tree_of(a, p, workspace);
  int status = AJQ_OK;
  with_dim(a->dim, [&](auto dim) {
    with_type(a->q_dtype, [&](auto q) {
      with_type(a->cache_dtype, [&](auto cache) {
        constexpr int HD = decltype(dim)::value;
        using QT = decltype(q);
        using CacheT = decltype(cache);
        auto launch = [&](auto kernel, int lds) {
          if ((status = allow_lds(kernel, lds, what)) != AJQ_OK) return;
          hipLaunchKernelGGL(kernel, dim3((unsigned)p.blocks), dim3(64 * p.waves), lds, (hipStream_t)stream, s);
          if ((status = check_launch(what)) != AJQ_OK || p.runs == 0) return;
          hipLaunchKernelGGL(tree_attention_merge_kernel<HD>, dim3((unsigned)ceil_div(p.queries, 4)), dim3(256), 0, (hipStream_t)stream, s);
          status = check_launch(what);
        };
        if constexpr (sizeof(CacheT) == 4) {
          if (p.walk) {
            auto laid = [&](auto tiles) {
              constexpr int RT = decltype(tiles)::value, lds = laid_lds_bytes<HD>();
              p.runs ? launch(tree_attention_laid_kernel<HD, QT, RT, false>, lds) : launch(tree_attention_laid_kernel<HD, QT, RT, true>, lds);
            };
            return p.rt == 2 ? laid(Size<2>{}) : laid(Size<1>{});
          }
        }
        if constexpr (sizeof(CacheT) == 2) {
          if (p.walk) {
            auto walk = [&](auto tiles) {
              constexpr int U = decltype(tiles)::value;
              if constexpr (HD >= 64) {
                if (p.waves == 8) return launch(tree_attention_walk_kernel<HD, QT, U, 8>, many_lds_bytes<HD, 8>());
              }
              launch(tree_attention_walk_kernel<HD, QT, U, 4>, many_lds_bytes<HD, 4>());
            };
            if constexpr (HD == 128 && sizeof(QT) == 2) {
              if (p.rt == 2) return walk(Size<2>{});
            }
            return walk(Size<1>{});
          }
        }
        auto few = [&](auto tiles, auto waves) {
          constexpr int RT = decltype(tiles)::value, WV = decltype(waves)::value, lds = some_lds_bytes<HD, CacheT, RT, WV>();
          if constexpr (sizeof(CacheT) == 2 || RT == 1 || WV == 8) {
            if (p.runs) return launch(tree_attention_few_kernel<HD, QT, CacheT, RT, WV, false>, lds);
          }
          launch(tree_attention_few_kernel<HD, QT, CacheT, RT, WV, true>, lds);
        };
        if constexpr (sizeof(CacheT) == 2 || HD < 128) {
          if (p.rt == 2 && p.waves == 8) return few(Size<2>{}, Size<8>{});
        }
        if (p.rt == 2) return few(Size<2>{}, Size<4>{});
        p.waves == 8 ? few(Size<1>{}, Size<8>{}) : few(Size<1>{}, Size<4>{});
      });
    });
  });
  return status;
}

int ajqt_keep_rows(const ajqt_keep_rows_args* a, void* stream) {
  const char* what = "ajqt_keep_rows";
  if (!a) return fail(AJQ_ERR_NULL, "%s: null arguments", what);
  if (!a->keys || !a->values || !a->rows || !a->index) return fail(AJQ_ERR_NULL, "%s: null pointer argument", what);
  if (!built_dim(a->dim)) return fail(AJQ_ERR_UNSUPPORTED, "%s: head size %d (128, 64 and 32 are built)", what, a->dim);
  if (!known(a->dtype)) return fail(AJQ_ERR_UNSUPPORTED, "%s: unknown element type", what);
  if (a->layers < 1 || a->batch < 1 || a->kv_heads < 1 || a->max_len < 1 || a->max_len > kMostRows || a->width < 1 || a->index_ld < 0 ||
      (a->batch > 1 && a->index_ld != 0 && a->index_ld < a->width))
    return fail(AJQ_ERR_SHAPE, "%s: unsupported shape (layers=%d batch=%d kv_heads=%d max_len=%d width=%d index_ld=%lld)", what, a->layers, a->batch,
                a->kv_heads, a->max_len, a->width, (long long)a->index_ld);
  if (a->cache_layer < 0 || a->cache_layer % 8 != 0) return fail(AJQ_ERR_ALIGN, "%s: the layers' stride must be a multiple of 8 elements", what);
  if (int e = check_caches(what, a->keys, a->values, a->cache_batch, a->cache_head)) return e;
  const long long size = a->dtype == AJQS_BF16 ? 2 : 4, row = a->dim * size;
  const long long apart = (long long)(reinterpret_cast<uintptr_t>(a->values) - reinterpret_cast<uintptr_t>(a->keys));
  Dimension dims[] = {{a->layers, a->cache_layer * size}, {a->batch, a->cache_batch * size}, {a->kv_heads, a->cache_head * size}, {2, std::abs(apart)}};
  if (!nested(dims, row * a->max_len)) return fail(AJQ_ERR_SHAPE, "%s: cache heads that overlap cannot be written", what);
  const long long heads = 2ll * a->layers * a->batch * a->kv_heads;
  // A short list's workgroup takes whole rows while they are four a lane, else a part of them.  A long list's are two a CU: where heads are fewer each takes a part of
  // the rows, of 128 bytes at least.
  const int all = (int)row / 16;
  int columns = 1;
  if (a->width > kShortList)
    while (columns * 8 < all && heads * columns < 512) columns *= 2;
  else
    while (a->width * all > 4 * 256 * columns) columns *= 2;
  const int lanes = all / columns, each = (a->width * lanes + 255) / 256;
  if (heads > kMostLanes / 1024 / columns || (double)a->layers * a->batch * a->kv_heads > 1e9)
    return fail(AJQ_ERR_SHAPE, "%s: %d x %d x %d heads", what, a->layers, a->batch, a->kv_heads);
  const KeepRows k{a->keys, a->values, int64s(a->rows), int64s(a->index), int64s(a->counts), int64s(a->offset), a->cache_layer, a->cache_batch,
                   a->cache_head, a->index_ld, a->max_len, a->width, (int)row, (int)size, lanes, divide_by(columns), divide_by(a->kv_heads), divide_by(a->batch)};
  const dim3 grid((unsigned)(heads * columns));
  if (a->width > kShortList) hipLaunchKernelGGL(keep_rows_kernel, grid, dim3(1024), 0, (hipStream_t)stream, k);
  else if (each > 2) hipLaunchKernelGGL(keep_path_kernel<4>, grid, dim3(256), 0, (hipStream_t)stream, k);
  else if (each > 1) hipLaunchKernelGGL(keep_path_kernel<2>, grid, dim3(256), 0, (hipStream_t)stream, k);
  else hipLaunchKernelGGL(keep_path_kernel<1>, grid, dim3(256), 0, (hipStream_t)stream, k);
  return check_launch(what);
}

size_t ajqt_log_probs_workspace(const ajqt_log_probs_args* a) { return check_log_probs(a) ? 0 : log_probs_plan(a).bytes; }

int ajqt_log_probs(const ajqt_log_probs_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "ajqt_log_probs";
  if (int e = check_log_probs(a)) return e;
  const LogProbsPlan p = log_probs_plan(a);
  if (a->rows * p.slices > kMostLanes / p.lanes) return fail(AJQ_ERR_SHAPE, "%s: %d rows of %d", what, a->rows, a->vocab);
  if (p.bytes && (!workspace || workspace_bytes < p.bytes))
    return fail(AJQ_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, p.bytes, workspace_bytes);
  if (!aligned16(workspace)) return fail(AJQ_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", what);
  f32x4_t* parts = reinterpret_cast<f32x4_t*>(workspace);
  unsigned long long* firsts = reinterpret_cast<unsigned long long*>(parts + (size_t)a->rows * p.slices);
  const LogProbs n{a->logits, int64s(a->targets), a->log_probs, a->entropy, a->top_log_probs, reinterpret_cast<long long*>(a->ranks),
                   reinterpret_cast<long long*>(a->top_ids), parts, reinterpret_cast<float*>(firsts + (size_t)a->rows * p.slices * a->top), firsts, a->ld, a->rows, a->vocab,
                   a->top, p.slice, (int)p.slices};
  with_type(a->dtype, [&](auto type) {
    using T = decltype(type);
    auto launch = [&](auto lanes, auto rank, auto top) {
      constexpr int LANES = decltype(lanes)::value;
      hipLaunchKernelGGL((log_probs_kernel<T, LANES, decltype(rank)::value, decltype(top)::value>), dim3((unsigned)(a->rows * p.slices)), dim3(LANES), 0,
                         (hipStream_t)stream, n);
    };
    const std::integral_constant<bool, true> yes;
    const std::integral_constant<bool, false> no;
    auto with_top = [&](auto lanes, auto rank) { a->top ? launch(lanes, rank, yes) : launch(lanes, rank, no); };
    auto with_rank = [&](auto lanes) { a->targets ? with_top(lanes, yes) : with_top(lanes, no); };
    p.lanes == 1024 ? with_rank(Size<1024>{}) : with_rank(Size<256>{});
  });
  if (int e = check_launch(what)) return e;
  if (p.slices == 1) return AJQ_OK;
  hipLaunchKernelGGL(log_probs_merge_kernel, dim3((unsigned)a->rows), dim3(a->top ? 256 : 64), 0, (hipStream_t)stream, n);
  return check_launch(what);
}

int ajqt_follow_drafts(const ajqt_follow_drafts_args* a, void* stream) {
  const char* what = "ajqt_follow_drafts";
  if (!a) return fail(AJQ_ERR_NULL, "%s: null arguments", what);
  if (!a->tokens || !a->parents || !a->choices || !a->path || !a->accepted || !a->chosen) return fail(AJQ_ERR_NULL, "%s: null pointer argument", what);
  if (a->batch < 1 || a->nodes < 1 || a->nodes > kMostNodes || a->tokens_ld < 0 || a->parents_ld < 0 || a->choices_ld < 0 || a->choices_step < 0 ||
      a->batch > kMostLanes / kFollowThreads)
    return fail(AJQ_ERR_SHAPE, "%s: unsupported shape (batch=%d nodes=%d, at most %d)", what, a->batch, a->nodes, kMostNodes);
  const FollowDrafts f{int64s(a->tokens), int64s(a->parents), int64s(a->choices), int64s(a->counts), reinterpret_cast<long long*>(a->path),
                       reinterpret_cast<long long*>(a->accepted), reinterpret_cast<long long*>(a->chosen), a->tokens_ld, a->parents_ld, a->choices_ld,
                       a->choices_step, a->nodes};
  hipLaunchKernelGGL(follow_drafts_kernel, dim3((unsigned)a->batch), dim3(kFollowThreads), 0, (hipStream_t)stream, f);
  return check_launch(what);
}

}  // extern "C"
