/*
 * minimax_paged.h — C ABI of a paged 8-bit key/value cache on B200: appending the new tokens of
 * several sequences with the rotary embedding applied on the way, and attention of those tokens
 * over the cache (single tokens, drafted tokens and prompt chunks in one call).
 *
 * No counterpart in the reference, whose cache is one sequence of f16 tensors
 * (src/model.rs:79-162); the rotary pairs, the head geometry and the softmax scale are its own
 * (partial_rope_f16, gqa_decode_f16_128), so a layer of the same weights attends alike.
 *
 * Pointers are device memory; the stream is a cudaStream_t handle; functions return an MMRS status
 * (minimax_moe.h).  Lengths, page numbers and row offsets are read on the device, so a captured
 * CUDA graph serves other lengths within the same bounds; host-side errors launch nothing.
 */
#ifndef MINIMAX_PAGED_H
#define MINIMAX_PAGED_H

#include "minimax_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MMRS_PAGED_HEAD_DIM 128
#define MMRS_PAGED_MAX_SEQS 1024 /* sequences a call takes                                      */
#define MMRS_PAGED_MAX_GROUP 16  /* query heads per KV head                                     */

/* Element types of queries, keys, values, outputs and logits. */
#define MMRS_TYPE_F32 0
#define MMRS_TYPE_F16 1
#define MMRS_TYPE_BF16 2

/* The cache of one layer.  A key (value) is its e4m3 code times the scale of its page and head.
 * Below a sequence's length value codes are finite; a key of NaN codes marks a token that was not
 * finite when it was appended.  Slots past the length may hold anything. */
typedef struct {
    void *k, *v;              /* e4m3 [num_pages][kv_heads][page_size][128], 128-byte aligned     */
    float *k_scale, *v_scale; /* f32 [num_pages][kv_heads], >= 0                                  */
    int num_pages;
    int page_size;            /* 16, 32, 64 or 128 positions                                      */
    int kv_heads;
} MmrsPagedCache;

/* The sequences of one call.  Sequence b brings the rows cu_q[b] .. cu_q[b + 1] - 1 of the call's
 * token rows; they are its last positions, seq_len[b] - (cu_q[b + 1] - cu_q[b]) .. seq_len[b] - 1.
 * Position j of it lies in slot j % page_size of page page_table[b][j / page_size]; a page number
 * outside [0, num_pages) holds nothing: appending to it writes nothing, attention does not see it.
 * max_q and max_len bound the device-side values (a sequence is cut to them). */
typedef struct {
    const int32_t *cu_q;       /* [num_seqs + 1], rising from 0                                   */
    const int32_t *seq_len;    /* [num_seqs], with this call's new tokens                         */
    const int32_t *page_table; /* [num_seqs][table_stride]                                        */
    int num_seqs;
    int table_stride;          /* max_len <= table_stride * page_size                             */
    int total_q;               /* token rows of the call                                          */
    int max_q;                 /* largest number of new tokens of a sequence                      */
    int max_len;               /* largest seq_len                                                 */
} MmrsPagedBatch;

/* Appends the batch's new tokens.  q [total_q][query_heads][128] and k, v [total_q][kv_heads][128]
 * of in_type, token rows q_stride (k_stride, v_stride) elements apart, 16-byte aligned; the first
 * rope_dim columns of every q and k head are rotated by the f32 tables rope_cos / rope_sin
 * [rope_positions][rope_dim / 2] at the token's position, pairs (i, i + rope_dim / 2), in f32:
 * (a, b) -> (a c - b s, b c + a s), each product and sum rounded once.  q_out [total_q][query_heads]
 * [128] of out_type (f16 or bf16) gets the rotated queries (q and q_out both null: keys and values
 * only).
 *   Scale of a page and head: the smallest power of two with |x| <= 448 scale for the page's new
 * tokens (at least 2^-64, 0 when they are all zero); a page that holds earlier tokens of the
 * sequence keeps its scale where that is larger, otherwise takes the new one and has its earlier
 * codes rounded again (exact but for e4m3 subnormals).  Codes round to nearest even.  A token whose
 * key or value of a head holds an infinity or NaN takes no part in the scales; its key there is
 * stored as NaN and its value as 0, so that every row that sees it becomes NaN and no other.
 * Calling it again with the same arguments leaves the cache as it is. */
MMRS_API int mmrs_paged_append(const MmrsPagedCache *cache, const MmrsPagedBatch *batch, const void *q, const void *k,
                               const void *v, int64_t q_stride, int64_t k_stride, int64_t v_stride, int in_type,
                               int query_heads, const float *rope_cos, const float *rope_sin, int rope_dim,
                               int rope_positions, void *q_out, int out_type, mmrs_stream_t stream);

/* Workspace bytes of mmrs_paged_attend for batches of at most num_seqs sequences and total_q token
 * rows (0: arguments out of range).  Caller-owned, 256-byte aligned, zero before first use; it
 * holds partial results and counters that every call leaves at zero.  One workspace serves one
 * stream at a time. */
MMRS_API size_t mmrs_paged_attend_workspace_bytes(int num_seqs, int total_q, int query_heads, int kv_heads);

/* Outcome of the completed calls on a workspace (synchronous read): MMRS_OK, or MMRS_ERR_TIMEOUT
 * when a bounded wait inside a kernel expired: the outputs of that call are incomplete.  The workspace
 * stays usable; its status word keeps the error until the caller zeroes it. */
MMRS_API int mmrs_paged_attend_status(const void *workspace);

/* Attention of the batch's token rows over the cache.  q [total_q][query_heads][128] of `type` (f16
 * or bf16, rows q_stride elements apart, 16-byte aligned); query head h reads KV head
 * h / (query_heads / kv_heads).  The row at position p sees the positions j <= p of its sequence and,
 * with window > 0, of those only p - j < window and j < sinks (the first tokens stay visible).
 * out [total_q][query_heads][128] of `type` = softmax(scale q k) v; lse f32 [total_q][query_heads]
 * (or null) = ln sum exp(scale q k).  A row that sees nothing gives 0 and -infinity.  Statistics
 * and sums are f32; probabilities are rounded to f16 for the second product, and bf16 queries go to f16
 * after a power-of-two scaling of their row (exact down to 2^-31 of its largest value).
 *   Value scales enter that product relative to a reference scale, rounded to f16 (exact for the powers
 * of two that the append writes), which follows the pages.  For a sequence of up to 48 rows a KV head
 * pages may lie 2^64 apart without values being lost next to larger ones.  For longer ones that holds
 * between runs of 128 positions (from a multiple of 128 on) up to 2^60; within one, values keep their
 * bits down to 2^-22 of its largest scale and lose them one by one below. */
MMRS_API int mmrs_paged_attend(const MmrsPagedCache *cache, const MmrsPagedBatch *batch, const void *q,
                               int64_t q_stride, int type, int query_heads, float scale, int window, int sinks,
                               void *out, float *lse, void *workspace, size_t workspace_bytes, mmrs_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* MINIMAX_PAGED_H */
