/*
 * iekv_ops.h — C-ABI of the operators that read the paged KV cache and score what
 * a model answers (libiekv_ops.so, MI355X / gfx950).
 *
 *   attention   of one layer of a step, read through block tables: sliding window
 *               with sink tokens, batches that share leading blocks
 *   microscaled caches: rows quantised as they are written, and read back as values
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

#define IEKV_OPS_ABI_VERSION 2

int iekv_ops_abi_version(void);

/* Message for the last failed call on this thread ("" if none). */
const char* iekv_ops_last_error(void);

/* Element types of caches only (beside IEKV_TYPE_*): microscaled. 32 dimensions of a head (the
 * last of a head may be fewer) share a power of two 2^e; an element x is held as x / 2^e rounded
 * to nearest even, in 8 bits (e4m3 of at most 448; integers of at most 127) or 4 (e2m1 of at
 * most 6; the even dimension in a byte's low half). e is the smallest from -100 on with which
 * the group's largest magnitude is within the type's. A head's record is the bytes of its
 * elements, then 4 bytes of which byte g is group g's e + 127 and those past the last group are
 * 0. A group with a NaN or an infinity has the byte 255, and its elements 0, and reads as NaN.
 * A cache is [num_blocks * block_size][num_kv_heads] records: rows like any other for the
 * handoff and whatever else moves bytes. */
enum { IEKV_TYPE_MXFP8 = 5, IEKV_TYPE_MXINT8 = 6, IEKV_TYPE_MXFP4 = 7 };

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
  int32_t cache_type;    /* the query type, _E4M3 or microscaled; any type for F32 queries.
                          * Microscaled elements are taken as the query type holds them */
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

/* Bytes of a record of head_dim dimensions (a multiple of 8 up to IEKV_ATTENTION_MAX_DIM):
 * head_dim + 4, or head_dim / 2 + 4 of MXFP4; 0 for any other type or size. */
int64_t iekv_mx_head_bytes(int32_t cache_type, int32_t head_dim);

/* What a pool's microscaled arrays have in common. */
typedef struct iekv_mx_cache {
  int32_t cache_type;   /* IEKV_TYPE_MX* */
  int32_t num_kv_heads, head_dim;
  int32_t block_size;   /* rows per block */
  int64_t num_blocks;
} iekv_mx_cache;

/* Quantise rows into slots, for n_layers layers: K and V of layer l and token t, the
 * num_kv_heads * head_dim values of row_type (F32, F16 or BF16) at k + l * k_strides[0] +
 * t * k_strides[1] + head * k_strides[2] elements (HOST arrays of three strides, head_dim
 * contiguous) and at v likewise, become the records of row slots[t] (int64, device memory) of
 * the arrays at k_arrays[l] and v_arrays[l] (HOST arrays of device addresses). Rows whose slot is
 * outside the pool are skipped; of rows with the same slot any may be held, or parts of several.
 * Runs on the current device, which has to be the arrays'. */
int iekv_mx_write_slots(const iekv_mx_cache* cache, const uint64_t* k_arrays,
                        const uint64_t* v_arrays, int32_t n_layers, int32_t row_type,
                        const void* k, const int64_t* k_strides, const void* v,
                        const int64_t* v_strides, const int64_t* slots, int64_t n_tokens,
                        hipStream_t stream);

/* The same with the slots in HOST memory: checked (IEKV_ERR_RANGE for one outside the pool), then
 * carried in the launches' own arguments, IEKV_MX_INLINE_SLOTS tokens per launch. */
#define IEKV_MX_INLINE_SLOTS 128
int iekv_mx_write_slots_ids(const iekv_mx_cache* cache, const uint64_t* k_arrays,
                            const uint64_t* v_arrays, int32_t n_layers, int32_t row_type,
                            const void* k, const int64_t* k_strides, const void* v,
                            const int64_t* v_strides, const int64_t* slots, int64_t n_tokens,
                            hipStream_t stream);

/* Read a context back as values: out [n_arrays][context_len][num_kv_heads][head_dim] of out_type
 * (F32, F16 or BF16; rounded to nearest even), row j of array i from the array at arrays[i]
 * (HOST array of device addresses), row table[j / block_size] * block_size + j % block_size
 * (int32, device memory). Rows of blocks outside the pool are left untouched. Runs on the
 * current device, which has to be the arrays'. */
int iekv_mx_read_rows(const iekv_mx_cache* cache, const uint64_t* arrays, int32_t n_arrays,
                      const int32_t* table, int64_t context_len, int32_t out_type, void* out,
                      hipStream_t stream);

/* The same with the table in HOST memory: checked (IEKV_ERR_RANGE for a used block outside the
 * pool), then carried in the launches' own arguments, IEKV_MX_INLINE_BLOCKS blocks per launch. */
#define IEKV_MX_INLINE_BLOCKS 256
int iekv_mx_read_rows_ids(const iekv_mx_cache* cache, const uint64_t* arrays, int32_t n_arrays,
                          const int32_t* table, int64_t context_len, int32_t out_type, void* out,
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
