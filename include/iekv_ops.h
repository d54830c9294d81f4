/*
 * iekv_ops.h — C-ABI of the operators that read the paged KV cache and score what
 * a model answers (libiekv_ops.so, MI355X / gfx950).
 *
 *   attention   of one layer of a step, read through block tables: sliding window
 *               with sink tokens, batches that share leading blocks
 *   logprobs    log probabilities of given tokens, entropy, most likely alternatives
 *
 * The conventions are those of iekv.h: IEKV_OK or a negative IEKV_ERR_* code, a
 * message per thread (iekv_ops_last_error), argument errors found before anything
 * is enqueued, work enqueued on the caller's stream, no allocation and no host
 * synchronization in the calls that enqueue. Element types are IEKV_TYPE_*.
 */
#ifndef IEKV_OPS_H_
#define IEKV_OPS_H_

#include <stdint.h>
#include <hip/hip_runtime_api.h>

#include "iekv.h"

#ifdef __cplusplus
extern "C" {
#endif

#define IEKV_OPS_ABI_VERSION 1

int iekv_ops_abi_version(void);

/* Message for the last failed call on this thread ("" if none). */
const char* iekv_ops_last_error(void);

#define IEKV_ATTENTION_MAX_DIM 128   /* largest head dimension (multiples of 8) */
#define IEKV_ATTENTION_MAX_GROUP 128 /* most query heads per KV head */
#define IEKV_ATTENTION_MAX_CONTEXT (1 << 30)

/* What the sequences of a step have in common. */
typedef struct iekv_attention_shape {
  int32_t num_heads;     /* query heads */
  int32_t num_kv_heads;  /* head h reads KV head h / (num_heads / num_kv_heads) */
  int32_t head_dim;
  int32_t block_size;    /* cache rows per block */
  int64_t num_blocks;    /* blocks of the pool (fewer than 2^32 rows): every table entry is below */
  int32_t query_type;    /* IEKV_TYPE_F32, _F16 or _BF16: of q and of the output */
  int32_t cache_type;    /* the query type, or _E4M3; any type for F32 queries */
  int64_t window;        /* a query sees the last `window` keys up to its own (0: all) */
  int64_t sinks;         /* and the first `sinks` keys */
  int64_t shared_blocks; /* leading blocks that every table shares: attended once for all where
                          * that saves more than joining the results takes */
} iekv_attention_shape;

/* How a step's attention is cut into workgroups: made once per step, used by every
 * layer. Holds no device memory. It is for the device that is current when it is made:
 * iekv_attend runs there, whatever device is current then. */
typedef struct iekv_attention_plan iekv_attention_plan;

/* Plan the attention of n_seqs sequences (HOST arrays). Sequence s has context_lens[s]
 * tokens in the cache, its queries are the last query_lens[s] of them, and its blocks
 * are tables[table_starts[s] .. table_starts[s+1]), of which the first
 * ceil(context / block_size) are used. Query i of s, at position
 * p = context - queries + i, sees the keys j <= p with j > p - window or j < sinks.
 * IEKV_ERR_RANGE for a used block outside the pool, IEKV_ERR_IDS for tables that do not
 * begin with the shared blocks. */
int iekv_attention_plan_create(const iekv_attention_shape* shape, int32_t n_seqs,
                               const int32_t* context_lens, const int32_t* query_lens,
                               const int32_t* tables, const int64_t* table_starts,
                               iekv_attention_plan** out);
int iekv_attention_plan_destroy(iekv_attention_plan* plan);

/* The plan's words (host memory of the plan's, to be copied to the device), how many
 * there are, the query rows of the step and the workspace iekv_attend needs. */
int iekv_attention_plan_info(const iekv_attention_plan* plan, const int32_t** words,
                             int64_t* n_words, int64_t* tokens, int64_t* workspace_bytes);

/* out[t][h] = softmax(scale * q[t][h] . K) V over the keys the row sees.
 * `words` is the device copy of the plan's words; k and v one layer's arrays
 * [num_blocks * block_size][num_kv_heads][head_dim]; q is [tokens][num_heads][head_dim]
 * with the given strides in elements (head_dim contiguous); out is contiguous, and may be
 * q itself where that is too, but not overlap it otherwise. The workspace is used until the
 * call's kernels end. */
int iekv_attend(const iekv_attention_plan* plan, const int32_t* words, const void* k,
                const void* v, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                float scale, void* out, void* workspace, int64_t workspace_bytes,
                hipStream_t stream);

#define IEKV_LOGPROBS_MAX_TOP 64

/* For each of n_rows rows x of `vocab` logits (row_stride elements apart) and its token t
 * (device int64): logprobs = x[t] - lse(x), entropy = -sum p ln p, and the `top` largest
 * logits in falling order, equal ones by index: top_logprobs [n_rows][top] = x - lse(x),
 * top_ids [n_rows][top]. Logits of -inf have probability zero. A row of nothing but -inf
 * has log probabilities of -inf and entropy 0; a row with a NaN or +inf has NaN log
 * probabilities and entropy (its alternatives put NaN first); a token outside 0..vocab-1
 * has log probability NaN. Runs on the current device, which has to be the arrays'. The
 * workspace (iekv_logprobs_workspace bytes, aligned to 16) is
 * used until the call's kernels end. */
int64_t iekv_logprobs_workspace(int32_t type, int64_t n_rows, int64_t vocab, int32_t top);
int iekv_logprobs(int32_t type, const void* logits, int64_t row_stride, int64_t n_rows,
                  int64_t vocab, const int64_t* tokens, int32_t top, float* logprobs,
                  float* entropy, float* top_logprobs, int64_t* top_ids, void* workspace,
                  int64_t workspace_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* IEKV_OPS_H_ */
