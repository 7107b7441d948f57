/*
 * ajq_draft -- operators of checking drafted tokens in one pass of the model, libajq_draft.so.
 *
 * A sequence has a cache [batch, kv_heads, max_len, dim] whose first rows[b] + *offset rows are committed.  A step takes `tokens`
 * tokens a sequence, a tree: token 0 (the last one chosen) is its root, the others are guesses of what follows.  Token t's keys and values lie in
 * row rows[b] + *offset + t, whatever its depth.  Attention lets each see the committed rows and its ancestors; the model's choices
 * decide which path through the tree was right; its rows move together and are committed.
 *
 * All pointers are device pointers unless said otherwise; calls are asynchronous on `stream`, allocate nothing and keep no
 * pointer.  Return value: 0 or a negative status as in ajq.h (ajqt_last_error() gives the calling thread's message).  What lies
 * on the device (rows, counts, parents, ids) is not seen by the host: the kernels hold it inside the buffers.  Element types:
 * AJQS_F32, AJQS_BF16 (ajq_serve.h).
 */
#ifndef AJQ_DRAFT_H
#define AJQ_DRAFT_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

const char* ajqt_last_error(void);

typedef struct {
  const void *q, *keys, *values;
  const uint32_t* masks;
  const int64_t *rows, *counts, *offset;
  void* out;
  int64_t cache_batch, cache_head, mask_batch, mask_token;
  int32_t batch, tokens, heads, kv_heads, dim, max_len;
  int32_t q_dtype, cache_dtype;
} ajqt_tree_attention_args;
/* out bf16 [batch, tokens, heads * dim] = softmax(q . k / sqrt(dim)) v of q [batch, heads, tokens, dim]: token t of sequence b sees the rows ahead
 * of rows[b] + *offset (offset NULL: 0) and, of the tokens' own, row rows[b] + *offset + u where bit u % 32 of word u / 32 of its mask is set and u <
 * counts[b] (NULL: all); none outside [0, max_len).  Masks: words of token t of sequence b at masks + b * mask_batch + t * mask_token
 * (mask_batch 0: one tree for all; at least (tokens + 31) / 32 words).  Zeros where a token is not there or sees nothing.  Values of the
 * committed rows and of the tokens that are there must be finite (one that is not may make its component NaN for all tokens of the sequence); rows behind
 * them may hold anything.  heads a multiple of kv_heads; dim 128, 64 or 32; caches fp32 or bf16, strides in elements, multiples of 8; q fp32 or bf16.
 *
 * Precision: sums, maxima and scores are fp32.  fp32 queries and rows enter the products as two bf16 numbers each (16 bits and more of them), and a weight is rounded
 * to bf16 ahead of the second product; but a call on fp32 rows that goes by tiles of 16 queries is in fp32 throughout (up to 16 queries of a key head always do, more of them
 * where that takes less time).  No atomics: the same bits from run to run, for one shape (which of the ways a call goes, and so its last bits, is chosen by batch,
 * tokens, heads, dim, max_len and types).
 *
 * Workspace (16-byte aligned; this call's alone until it is done): what the first function says.  0 bytes where every sequence's rows are walked in one part; else
 * 8 a sequence and tokens * heads * (4 * dim + 8) a part, for up to 64 parts a sequence and 1024 / kv_heads in all. */
size_t ajqt_tree_attention_workspace(const ajqt_tree_attention_args* args);
int ajqt_tree_attention(const ajqt_tree_attention_args* args, void* workspace, size_t workspace_bytes, void* stream);

typedef struct {
  void *keys, *values;
  const int64_t *rows, *index, *counts, *offset;
  int64_t cache_layer, cache_batch, cache_head, index_ld;
  int32_t layers, batch, kv_heads, dim, max_len, width;
  int32_t dtype;
} ajqt_keep_rows_args;
/* In each of the layers' caches (strides in elements, multiples of 8; no two heads may overlap) row rows[b] + *offset + i becomes what row rows[b] +
 * *offset + index[b * index_ld + i] was, i = 0 .. min(counts[b], width) - 1 (counts NULL: width).  A list goes on while its numbers ascend from
 * 0 or more and their rows are in the cache: it ends ahead of the first that does not (and a sequence whose rows begin outside [0, max_len) has none).  No
 * other row is written. */
int ajqt_keep_rows(const ajqt_keep_rows_args* args, void* stream);

typedef struct {
  const void* logits;
  const int64_t* targets;
  float *log_probs, *entropy, *top_log_probs;
  int64_t *ranks, *top_ids;
  int64_t ld;
  int32_t rows, vocab, top, dtype;
} ajqt_log_probs_args;
/* Of each row x of logits [rows, vocab] (fp32 or bf16, row stride ld; a token's probability is p_v = exp(x_v) / sum exp(x)):
 *   entropy[r] = - sum p_v log p_v
 *   log_probs[r] = log p_t, ranks[r] = how many tokens have a larger logit than t, or the same one and a smaller id   (t = targets[r]; targets NULL: neither;
 *                  0 and -1 for a t outside [0, vocab))
 *   top_ids, top_log_probs [rows, top]: the first `top` tokens in that order (0: neither; at most 64, and vocab).
 * A row of -inf only: -inf throughout, entropy 0.  A row with NaN or +inf: NaN, and some numbers inside [0, vocab).
 * All sums in fp32.  Workspace (16-byte aligned): what the first function says.  0 where a row is at most 32768 fp32 or 65536 bf16 logits (the 16 bytes that an unaligned
 * row begins in less); else 4 bytes a row and 16 + 8 * top for each of its slices, of that size at most or, of few rows, a quarter of it. */
size_t ajqt_log_probs_workspace(const ajqt_log_probs_args* args);
int ajqt_log_probs(const ajqt_log_probs_args* args, void* workspace, size_t workspace_bytes, void* stream);

typedef struct {
  const int64_t *tokens, *parents, *choices, *counts;
  int64_t *path, *accepted, *chosen;
  int64_t tokens_ld, parents_ld, choices_ld, choices_step;
  int32_t batch, nodes;
} ajqt_follow_drafts_args;
/* Trees of nodes [batch, nodes]: node 0 is the root, node t > 0 a child of parents[t] (in [0, t); a node with another parent is in no tree) that
 * guesses tokens[t]; choices[t] (elements choices_step apart) is the model's choice behind node t.  From the root on, each step goes to the first child
 * whose guess is the choice behind the node it is at; the first counts[b] (NULL: all) nodes are there.
 *   accepted[b]  how many nodes the path has (the root is one; 0 where it is not there)
 *   path [batch, nodes]    the path's nodes, ascending, then -1
 *   chosen [batch, nodes]  the choices behind them, then -1: the tokens that the step has produced
 * parents_ld may be 0: one tree for all.  At most 4096 nodes. */
int ajqt_follow_drafts(const ajqt_follow_drafts_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* AJQ_DRAFT_H */
