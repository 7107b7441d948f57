// C ABI of libajq_serve.so (include/ajq_serve.h): argument validation, launch geometry, error reporting.
#include <algorithm>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include "../../include/ajq_serve.h"
#include "ajq_common.h"
#include "logits_kernels.h"
#include "norm_rope_kernels.h"
#include "shared_attention.h"

using namespace ajq;

namespace {

thread_local char g_error[512] = "";

int fail(int status, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, ap);
  va_end(ap);
  return status;
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
bool known(int dtype) { return dtype == AJQS_BF16 || dtype == AJQS_F32; }
int check_launch(const char* what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(AJQ_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
  return AJQ_OK;
}
const long long* int64s(const int64_t* p) { return reinterpret_cast<const long long*>(p); }

// Calls fn(T{}) for the element type of a dtype flag.
template <typename F>
void with_type(int dtype, F&& fn) {
  if (dtype == AJQS_BF16) fn(uint16_t{});
  else fn(float{});
}
template <int N> struct Size {
  static constexpr int value = N;
};
template <typename F>
void with_dim(int dim, F&& fn) {
  if (dim == 128) fn(Size<128>{});
  else if (dim == 64) fn(Size<64>{});
  else fn(Size<32>{});
}
bool built_dim(int dim) { return dim == 128 || dim == 64 || dim == 32; }

int check_caches(const char* what, const void* keys, const void* values, long long outer, long long head) {
  if (!aligned16(keys) || !aligned16(values) || outer % 8 != 0 || head % 8 != 0)
    return fail(AJQ_ERR_ALIGN, "%s: caches must be 16-byte aligned, their strides multiples of 8 elements", what);
  if (outer < 0 || head < 0) return fail(AJQ_ERR_SHAPE, "%s: negative cache stride", what);
  return AJQ_OK;
}

int check_shared(const ajqs_shared_attention_args* a) {
  const char* what = "ajqs_shared_attention";
  if (!a) return fail(AJQ_ERR_NULL, "%s: null arguments", what);
  if (!a->q || !a->prefix_keys || !a->prefix_values || !a->keys || !a->values || !a->prefix_lengths || !a->rows || !a->out)
    return fail(AJQ_ERR_NULL, "%s: null pointer argument", what);
  if (!built_dim(a->dim)) return fail(AJQ_ERR_UNSUPPORTED, "%s: head size %d (128, 64 and 32 are built)", what, a->dim);
  if (a->batch < 1 || a->tokens < 1 || a->groups < 1 || a->batch % a->groups != 0 || a->kv_heads < 1 || a->heads < 1 ||
      a->heads % a->kv_heads != 0 || a->prefix_cap < 1 || a->max_len < 1)
    return fail(AJQ_ERR_SHAPE, "%s: unsupported shape (groups=%d batch=%d tokens=%d heads=%d kv_heads=%d prefix_cap=%d max_len=%d)", what,
                a->groups, a->batch, a->tokens, a->heads, a->kv_heads, a->prefix_cap, a->max_len);
  if ((long long)a->batch * a->heads * a->tokens > 0x1FFFFFFFLL)
    return fail(AJQ_ERR_SHAPE, "%s: too many queries (%d x %d x %d)", what, a->batch, a->heads, a->tokens);
  if (!known(a->q_dtype) || !known(a->cache_dtype)) return fail(AJQ_ERR_UNSUPPORTED, "%s: unknown element type", what);
  if (!aligned16(a->q) || !aligned16(a->out)) return fail(AJQ_ERR_ALIGN, "%s: q and out must be 16-byte aligned", what);
  if (int e = check_caches(what, a->prefix_keys, a->prefix_values, a->prefix_group, a->prefix_head)) return e;
  return check_caches(what, a->keys, a->values, a->cache_batch, a->cache_head);
}

SharedAttention shared_of(const ajqs_shared_attention_args* a) {
  return SharedAttention{a->q, a->prefix_keys, a->prefix_values, a->keys, a->values, int64s(a->prefix_lengths), int64s(a->rows),
                         int64s(a->counts), int64s(a->offset), reinterpret_cast<uint16_t*>(a->out), a->prefix_group, a->prefix_head,
                         a->cache_batch, a->cache_head, a->groups, a->batch, a->tokens, a->heads, a->kv_heads, a->prefix_cap, a->max_len,
                         kLog2e / sqrtf((float)a->dim)};
}

}  // namespace

extern "C" {

const char* ajqs_last_error(void) { return g_error; }

int ajqs_norm_rope(const ajqs_norm_rope_args* a, void* stream) {
  const char* what = "ajqs_norm_rope";
  if (!a) return fail(AJQ_ERR_NULL, "%s: null arguments", what);
  if (!a->qkv || !a->cosine || !a->sine || !a->rows || !a->keys || !a->values || !a->q)
    return fail(AJQ_ERR_NULL, "%s: null pointer argument", what);
  if (!built_dim(a->dim)) return fail(AJQ_ERR_UNSUPPORTED, "%s: head size %d (128, 64 and 32 are built)", what, a->dim);
  if (a->batch < 1 || a->tokens < 1 || a->kv_heads < 1 || a->heads < 1 || a->heads % a->kv_heads != 0 || a->max_len < 1 || a->table_rows < 1 ||
      (long long)a->batch * a->tokens > 0x7FFFFFFFLL)
    return fail(AJQ_ERR_SHAPE, "%s: unsupported shape (batch=%d tokens=%d heads=%d kv_heads=%d max_len=%d table_rows=%d)", what, a->batch,
                a->tokens, a->heads, a->kv_heads, a->max_len, a->table_rows);
  const long long all = (long long)a->heads + 2ll * a->kv_heads, room = (long long)a->max_len * a->dim;
  if (all > 1 << 20 || a->ld < all * a->dim || a->ld % 4 != 0)
    return fail(AJQ_ERR_SHAPE, "%s: rows of %lld elements (a multiple of 4, at least %lld)", what, (long long)a->ld, all * a->dim);
  if (!known(a->in_dtype) || !known(a->q_dtype) || !known(a->cache_dtype)) return fail(AJQ_ERR_UNSUPPORTED, "%s: unknown element type", what);
  if (!aligned16(a->qkv) || !aligned16(a->q) || !aligned16(a->cosine) || !aligned16(a->sine) || !aligned16(a->q_gain) || !aligned16(a->k_gain))
    return fail(AJQ_ERR_ALIGN, "%s: qkv, q, the tables and the gains must be 16-byte aligned", what);
  if (int e = check_caches(what, a->keys, a->values, a->cache_batch, a->cache_head)) return e;
  if ((a->kv_heads > 1 && a->cache_head < room) || (a->batch > 1 && a->cache_batch < room))
    return fail(AJQ_ERR_SHAPE, "%s: cache heads that overlap cannot be written", what);
  const NormRope n{a->qkv, a->cosine, a->sine, a->q_gain, a->k_gain, int64s(a->rows), int64s(a->positions), int64s(a->counts),
                   int64s(a->offset), a->keys, a->values, a->q, a->ld, a->cache_batch, a->cache_head, a->tokens, a->heads, a->kv_heads,
                   a->max_len, a->table_rows, a->eps};
  with_dim(a->dim, [&](auto dim) {
    with_type(a->in_dtype, [&](auto in) {
      with_type(a->q_dtype, [&](auto q) {
        with_type(a->cache_dtype, [&](auto cache) {
          constexpr int U = 1;
          const dim3 grid((unsigned)(a->batch * a->tokens), (unsigned)((all + 16 * U - 1) / (16 * U)));
          hipLaunchKernelGGL((norm_rope_kernel<decltype(in), decltype(q), decltype(cache), decltype(dim)::value, U>), grid, dim3(256), 0,
                             (hipStream_t)stream, n);
        });
      });
    });
  });
  return check_launch(what);
}

size_t ajqs_shared_attention_workspace(const ajqs_shared_attention_args* a) { return check_shared(a) ? 0 : 0; }

int ajqs_shared_attention(const ajqs_shared_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "ajqs_shared_attention";
  if (int e = check_shared(a)) return e;
  const size_t need = ajqs_shared_attention_workspace(a);
  if (need && (!workspace || workspace_bytes < need))
    return fail(AJQ_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, need, workspace_bytes);
  if (!aligned16(workspace)) return fail(AJQ_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", what);
  const SharedAttention s = shared_of(a);
  const long long queries = (long long)a->batch * a->heads * a->tokens;
  with_dim(a->dim, [&](auto dim) {
    with_type(a->q_dtype, [&](auto q) {
      with_type(a->cache_dtype, [&](auto cache) {
        hipLaunchKernelGGL((shared_attention_plain_kernel<decltype(q), decltype(cache), decltype(dim)::value>), dim3((unsigned)((queries + 3) / 4)),
                           dim3(256), 0, (hipStream_t)stream, s);
      });
    });
  });
  return check_launch(what);
}

int ajqs_adjust_logits(const ajqs_adjust_logits_args* a, void* stream) {
  const char* what = "ajqs_adjust_logits";
  if (!a) return fail(AJQ_ERR_NULL, "%s: null arguments", what);
  if (!a->logits || !a->out || (a->bias_ids && !a->bias)) return fail(AJQ_ERR_NULL, "%s: null pointer argument", what);
  if (a->batch < 1 || a->vocab < 1 || a->ld < a->vocab || a->out_ld < a->vocab)
    return fail(AJQ_ERR_SHAPE, "%s: unsupported shape (batch=%d vocab=%d ld=%lld out_ld=%lld)", what, a->batch, a->vocab, (long long)a->ld,
                (long long)a->out_ld);
  if (!known(a->dtype)) return fail(AJQ_ERR_UNSUPPORTED, "%s: unknown element type", what);
  if (a->logits == a->out && (a->dtype != AJQS_F32 || a->ld != a->out_ld))
    return fail(AJQ_ERR_UNSUPPORTED, "%s: only fp32 logits can be adjusted in place, row by row", what);
  if (a->tokens && (a->max_tokens < 0 || a->max_tokens > kMaxHistory || a->tokens_ld < a->max_tokens))
    return fail(AJQ_ERR_SHAPE, "%s: %d tokens a row (at most %d, and the rows' stride %lld)", what, a->max_tokens, kMaxHistory,
                (long long)a->tokens_ld);
  if (a->prompt && (a->max_prompt < 0 || a->max_prompt > kMaxHistory || a->prompt_ld < a->max_prompt))
    return fail(AJQ_ERR_SHAPE, "%s: %d prompt tokens a row (at most %d, and the rows' stride %lld)", what, a->max_prompt, kMaxHistory,
                (long long)a->prompt_ld);
  if (a->bias_ids && (a->biases < 0 || a->biases > kMaxBiases || a->bias_ld < a->biases))
    return fail(AJQ_ERR_SHAPE, "%s: %d biases a row (at most %d, and the rows' stride %lld)", what, a->biases, kMaxBiases, (long long)a->bias_ld);
  if (a->allowed && (a->masks < 1 || a->allowed_ld < ((long long)a->vocab + 31) / 32))
    return fail(AJQ_ERR_SHAPE, "%s: masks of %lld words for a vocabulary of %d", what, (long long)a->allowed_ld, a->vocab);
  if (a->allowed && !a->allowed_rows && a->masks < a->batch)
    return fail(AJQ_ERR_SHAPE, "%s: %d masks for %d rows", what, a->masks, a->batch);
  if (!aligned4(a->out) || !aligned4(a->allowed) || (a->dtype == AJQS_F32 && !aligned4(a->logits)) || (reinterpret_cast<uintptr_t>(a->logits) & 1u))
    return fail(AJQ_ERR_ALIGN, "%s: logits, out and the masks must be aligned to their elements", what);
  const int slice = 8192;
  AdjustLogits n{a->logits, a->out, int64s(a->tokens), int64s(a->token_counts), int64s(a->prompt), int64s(a->prompt_counts), a->repetition,
                 a->frequency, a->presence, int64s(a->bias_ids), a->bias, a->allowed, int64s(a->allowed_rows), a->ld, a->out_ld, a->tokens_ld,
                 a->prompt_ld, a->bias_ld, a->allowed_ld, a->vocab, a->max_tokens, a->max_prompt, a->bias_ids ? a->biases : 0, a->masks,
                 a->token_count_stride, a->prompt_count_stride, slice};
  const long long slices = ((long long)a->vocab + slice - 1) / slice;
  if (slices > 65535) return fail(AJQ_ERR_SHAPE, "%s: vocabulary of %d", what, a->vocab);
  const bool words = (a->tokens && a->max_tokens) || (a->prompt && a->max_prompt) || n.biases;
  with_type(a->dtype, [&](auto type) {
    if (words)
      hipLaunchKernelGGL((adjust_logits_kernel<decltype(type), true>), dim3(a->batch, (unsigned)slices), dim3(1024), slice * 4, (hipStream_t)stream, n);
    else
      hipLaunchKernelGGL((adjust_logits_kernel<decltype(type), false>), dim3(a->batch, (unsigned)slices), dim3(1024), 0, (hipStream_t)stream, n);
  });
  return check_launch(what);
}

}  // extern "C"
