// C ABI of libajq_draft.so (include/ajq_draft.h): argument validation, launch geometry, error reporting.
#include "serve_host.h"

#include "../../include/ajq_draft.h"
#include "draft_kernels.h"
#include "log_probs_kernels.h"
#include "tree_attention.h"
#include "tree_plan.h"

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
