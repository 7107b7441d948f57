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

}  // namespace

extern "C" {

const char* ajqt_last_error(void) { return g_error; }

size_t ajqt_tree_attention_workspace(const ajqt_tree_attention_args* a) { return check_tree(a) ? 0 : 0; }

int ajqt_tree_attention(const ajqt_tree_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "ajqt_tree_attention";
  if (int e = check_tree(a)) return e;
  if (a->heads > 0xFFFF || a->batch > 0xFFFF) return fail(AJQ_ERR_SHAPE, "%s: %d heads of %d sequences", what, a->heads, a->batch);
  const TreeAttention s{a->q, a->keys, a->values, a->masks, int64s(a->rows), int64s(a->counts), int64s(a->offset), reinterpret_cast<uint16_t*>(a->out),
                        a->cache_batch, a->cache_head, a->mask_batch, a->mask_token, a->batch, a->tokens, a->heads, a->kv_heads, a->max_len,
                        kLog2e / sqrtf((float)a->dim)};
  with_dim(a->dim, [&](auto dim) {
    with_type(a->q_dtype, [&](auto q) {
      with_type(a->cache_dtype, [&](auto cache) {
        hipLaunchKernelGGL((tree_attention_kernel<decltype(dim)::value, decltype(q), decltype(cache)>),
                           dim3((unsigned)a->tokens, (unsigned)a->heads, (unsigned)a->batch), dim3(64), 0, (hipStream_t)stream, s);
      });
    });
  });
  return check_launch(what);
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
  const long long blocks = 2ll * a->layers * a->batch * a->kv_heads;
  if (blocks > kMostLanes / 1024 || (double)a->layers * a->batch * a->kv_heads > 1e9) return fail(AJQ_ERR_SHAPE, "%s: %d x %d x %d heads", what, a->layers, a->batch, a->kv_heads);
  const KeepRows k{a->keys, a->values, int64s(a->rows), int64s(a->index), int64s(a->counts), int64s(a->offset), a->cache_layer, a->cache_batch,
                   a->cache_head, a->index_ld, a->batch, a->kv_heads, a->max_len, a->width, (int)row, (int)size};
  hipLaunchKernelGGL(keep_rows_kernel, dim3((unsigned)blocks), dim3(a->width <= 64 ? 256 : 1024), 0, (hipStream_t)stream, k);
  return check_launch(what);
}

size_t ajqt_log_probs_workspace(const ajqt_log_probs_args*) { return 0; }

int ajqt_log_probs(const ajqt_log_probs_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "ajqt_log_probs";
  if (!a) return fail(AJQ_ERR_NULL, "%s: null arguments", what);
  if (!a->logits || (a->targets && (!a->log_probs || !a->ranks)) || (a->top && (!a->top_log_probs || !a->top_ids)))
    return fail(AJQ_ERR_NULL, "%s: null pointer argument", what);
  if (!known(a->dtype)) return fail(AJQ_ERR_UNSUPPORTED, "%s: unknown element type", what);
  if (a->rows < 1 || a->vocab < 1 || a->ld < 0 || a->top < 0 || a->top > kMostTop || a->top > a->vocab)
    return fail(AJQ_ERR_SHAPE, "%s: unsupported shape (rows=%d vocab=%d ld=%lld top=%d)", what, a->rows, a->vocab, (long long)a->ld, a->top);
  if (!aligned4(a->log_probs) || !aligned4(a->entropy) || !aligned4(a->top_log_probs) || (a->dtype == AJQS_F32 && !aligned4(a->logits)) ||
      (reinterpret_cast<uintptr_t>(a->logits) & 1u))
    return fail(AJQ_ERR_ALIGN, "%s: logits and results must be aligned to their elements", what);
  if (a->rows > kMostLanes / 256) return fail(AJQ_ERR_SHAPE, "%s: %d rows in a launch", what, a->rows);
  const LogProbs n{a->logits, int64s(a->targets), a->log_probs, a->entropy, a->top_log_probs, reinterpret_cast<long long*>(a->ranks),
                   reinterpret_cast<long long*>(a->top_ids), a->ld, a->rows, a->vocab, a->top};
  with_type(a->dtype, [&](auto type) {
    hipLaunchKernelGGL(log_probs_kernel<decltype(type)>, dim3((unsigned)a->rows), dim3(256), 0, (hipStream_t)stream, n);
  });
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
