/*
 * ajq_serve -- operators of decoding many continuations of one prompt, libajq_serve.so.
 *
 * A batch's sequences are at positions of their own.  Each has a cache of its own rows [batch, kv_heads, max_len, dim]; where
 * they share a first part (an instruction, a document, the prompt that they all complete) its rows lie once, in caches
 * [groups, kv_heads, prefix_cap, dim], for the batch / groups consecutive sequences of a group.
 *
 * All pointers are device pointers unless said otherwise; calls are asynchronous on `stream`, allocate nothing and keep no
 * pointer.  Return value: 0 or a negative status as in ajq.h (ajqs_last_error() gives the calling thread's message).  What lies
 * on the device (rows, counts, lengths, token ids) is not seen by the host: the kernels hold it inside the buffers.
 *
 * The first of a sequence's `tokens` new tokens takes row rows[b] + *offset of its own cache, the next ones the rows behind;
 * counts[b] (NULL: all) of the tokens are there.  `offset` (int64, NULL: 0) is one number for the batch, so that a recorded
 * graph can be replayed while a step counter on the device moves.
 */
#ifndef AJQ_SERVE_H
#define AJQ_SERVE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define AJQS_F32 0
#define AJQS_BF16 1

const char* ajqs_last_error(void);

typedef struct {
  const void* qkv;
  const float *cosine, *sine, *q_gain, *k_gain;
  const int64_t *rows, *positions, *counts, *offset;
  void *keys, *values, *q;
  int64_t ld, cache_batch, cache_head;
  int32_t batch, tokens, heads, kv_heads, dim, max_len, table_rows;
  int32_t in_dtype, q_dtype, cache_dtype;
  float eps;
} ajqs_norm_rope_args;
/* Projection rows qkv [batch * tokens, ld] = (heads query heads | kv_heads key heads | kv_heads value heads) of `dim`: every query and
 * key head x becomes x / sqrt(mean(x^2) + eps) * gain (q_gain, k_gain fp32 [dim]; NULL: as it is), then its pairs (x[2i], x[2i + 1])
 * turn by the tables' row positions[b] + *offset + t (positions NULL: rows; cosine, sine fp32 [table_rows, dim / 2]; held inside the
 * tables).  Queries go to q [batch, heads, tokens, dim] (zeros where a token is not there), keys and values to the token's row of the caches
 * (element strides cache_batch, cache_head); a row outside [0, max_len) is not written.  dim 128, 64 or 32;
 * no head of the caches may overlap another.
 * (RMSNorm.forward, src/ajllm/modeling/layers.py:70-74, on each head; RotaryPositionalEmbedding.forward, attention.py:36-60.) */
int ajqs_norm_rope(const ajqs_norm_rope_args* args, void* stream);

typedef struct {
  const void *q, *prefix_keys, *prefix_values, *keys, *values;
  const int64_t *prefix_lengths, *rows, *counts, *offset;
  void* out;
  int64_t prefix_group, prefix_head, cache_batch, cache_head;
  int32_t groups, batch, tokens, heads, kv_heads, dim, prefix_cap, max_len;
  int32_t q_dtype, cache_dtype;
} ajqs_shared_attention_args;
/* out bf16 [batch, tokens, heads * dim] = softmax(q . k / sqrt(dim)) v of q [batch, heads, tokens, dim]: token t of sequence b sees the
 * first prefix_lengths[g] rows (at most prefix_cap; g = b / (batch / groups)) of its group's prefix caches and its own rows 0 ..
 * rows[b] + *offset + t (at most max_len), which hold the new tokens already.  Zeros where a token is not there or sees nothing.  Values
 * that a token of the sequence sees must be finite (one that is not may make its component NaN for all tokens of the call, earlier ones too);
 * rows that no token of a sequence sees may hold anything.  heads a
 * multiple of kv_heads; dim 128, 64 or 32; caches fp32 or bf16, strides in elements, multiples of 8; q fp32 or bf16.
 * Products carry all bits of bf16 caches and queries and sixteen at least of fp32 ones; a weight is rounded to bf16 for its product with the values, but
 * for fp32 rows that tiles of 16 queries meet (short runs; at most 16, or 32, queries of a key head), which are in fp32 throughout; sums, maxima and denominators are fp32.
 * How the call is cut up goes by the capacities prefix_cap and max_len, since the lengths are on the device: choose them near to what will be filled.  The
 * workspace holds [parts, batch * heads * tokens] of dim + 2 fp32 numbers; on fp32 caches two parts at least of all but short runs, whatever the number of
 * tokens (1.06 GB for 16 x 2000 tokens of 32 heads of 128 behind 2048 rows), on bf16 ones none where more than 64 queries of a sequence and key head make tiles enough.
 * (scaled_dot_product_attention, src/ajllm/modeling/attention.py:20-33.) */
size_t ajqs_shared_attention_workspace(const ajqs_shared_attention_args* args);
int ajqs_shared_attention(const ajqs_shared_attention_args* args, void* workspace, size_t workspace_bytes, void* stream);

typedef struct {
  const void* logits;
  float* out;
  const int64_t *tokens, *token_counts, *prompt, *prompt_counts;
  const float *repetition, *frequency, *presence;
  const int64_t* bias_ids;
  const float* bias;
  const uint32_t* allowed;
  const int64_t* allowed_rows;
  int64_t ld, out_ld, tokens_ld, prompt_ld, bias_ld, allowed_ld;
  int32_t batch, vocab, max_tokens, max_prompt, biases, masks, token_count_stride, prompt_count_stride;
  int32_t dtype;
} ajqs_adjust_logits_args;
/* out[b, v] (fp32, row stride out_ld; may be the fp32 logits themselves, and overlap them in no other way) from x = logits[b, v] (dtype, row stride ld):
 *   x > 0 ? x / repetition[b] : x * repetition[b]   where v is among row b's prompt or tokens;
 *   x - (frequency[b] * n + presence[b])            where v is n > 0 times among its tokens;
 *   x + the sum of bias[b, i] over bias_ids[b, i] == v, in the order of i;
 *   -inf                                            where bit v % 32 of word v / 32 of its mask is clear.
 * The first min(token_counts[b * token_count_stride], max_tokens) of row b's tokens count (stride 0: one number for all; token_counts
 * NULL: all), prompt likewise.  Ids outside [0, vocab) are passed over.  Mask of row b: row allowed_rows[b] of allowed [masks, allowed_ld] (NULL: row b),
 * none where that is not in [0, masks).  Each of repetition, frequency and presence may be NULL (1, 0, 0), as may
 * tokens, prompt, bias_ids and allowed.  Row strides of tokens, prompt and allowed may be 0: one list, or mask, for all rows.  Up to 1024 biases a
 * row, 1048575 tokens a row. */
int ajqs_adjust_logits(const ajqs_adjust_logits_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* AJQ_SERVE_H */
