/*
 * minimax_sample.h — C ABI of token sampling over a decode step's logits on B200: greedy,
 * top-k, top-p (nucleus) and temperature sampling, and the log-probability of one token, all on
 * the device that holds the logits (no vocabulary-sized copy to the host).
 *
 * Reference: src/sampling.rs (TokenSampler::sample, :84-150; exponential_weights, :161-177;
 * compare_candidates, :154-159; token_logprob, :60-75; SamplingParams::validate, :31-39).  The
 * reference draws its random number from a per-request StdRng (`rng.random::<f64>()`, one draw
 * per stochastic sample); here the caller keeps that generator and passes the draw as `u`, so
 * the GPU choice for a given draw is the reference's choice.
 *
 * Pointers are device memory; the stream is a cudaStream_t handle.  Status codes as in
 * minimax_moe.h.  The workspace is caller-owned, 256-byte aligned and zero before first use;
 * every completed call leaves it ready for the next one (a call that ended in MMRS_ERR_TIMEOUT
 * leaves it to be zeroed again).  One workspace serves one stream at a time.
 */
#ifndef MINIMAX_SAMPLE_H
#define MINIMAX_SAMPLE_H

#include "minimax_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MMRS_ERR_NONFINITE 7 /* logits (or the log-probability) not finite: no token written   */

/* SamplingParams (src/sampling.rs:13-17).  Valid: temperature finite and >= 0, top_p finite in
 * [0, 1] (validate, :31-39); top_k 0 = no top-k cut. */
typedef struct {
    double temperature;
    double top_p;
    int top_k;
} MmrsSamplingParams;

/* Largest vocabulary a call takes (token ids fit 20 bits). */
#define MMRS_SAMPLE_MAX_VOCAB 1048576
/* Largest candidate set that top-p sorts: min(top_k, vocab) when top_k > 0, else the nucleus
 * itself.  A larger nucleus ends in MMRS_ERR_UNSUPPORTED (device status, token -1). */
#define MMRS_SAMPLE_MAX_SORTED 1024

/* Workspace bytes of mmrs_sample_token / mmrs_token_logprob for this vocabulary (0: vocabulary
 * out of range). */
MMRS_API size_t mmrs_sample_workspace_bytes(int vocab);

/* Outcome of the last completed call on a workspace (synchronous read): MMRS_OK,
 * MMRS_ERR_NONFINITE, MMRS_ERR_UNSUPPORTED (nucleus over MMRS_SAMPLE_MAX_SORTED) or
 * MMRS_ERR_TIMEOUT (a grid barrier's bounded wait expired). */
MMRS_API int mmrs_sample_workspace_status(const void *workspace);

/* No single counterpart in the reference: TokenSampler::sample (src/sampling.rs:84-150) with the
 * draw `u` = rng.random::<f64>() in [0, 1) supplied by the caller.  logits f32 [vocab]; token
 * int32 (device memory) = the chosen id, or -1 when the device status is not MMRS_OK.
 *   temperature 0: the first index of the largest logit (logits.argmax, :87-89; no finiteness
 *     check, as the reference).
 *   otherwise: non-finite logits -> MMRS_ERR_NONFINITE (:97-99); candidates = the top_k largest
 *     (logit descending, then id ascending: compare_candidates); with top_p < 1 and more than one
 *     candidate, the sorted candidates are cut after the first whose cumulative weight
 *     exp(l - max) reaches top_p of the total (:110-125); then one candidate is drawn with weights
 *     exp((l - max) / temperature) by walking the cumulative weights against u * total (:127-150).
 *     Without the top-p cut the walk visits candidates by ascending id (the reference's order when
 *     top_k is 0 or >= vocab; for 0 < top_k < vocab the reference walks in the order its
 *     partial selection left, which no caller can observe except through the draw).
 * Host-side errors (MMRS_ERR_ARG: null pointers, vocab out of range, invalid params, u outside
 * [0, 1), short workspace) launch nothing. */
MMRS_API int mmrs_sample_token(const float *logits, int vocab, const MmrsSamplingParams *params, double u,
                               int32_t *token, void *workspace, size_t workspace_bytes, mmrs_stream_t stream);

/* token_logprob (src/sampling.rs:60-75): out (f32, device memory) = ln softmax(logits)[token_id]
 * over the unfiltered distribution, accumulated in double.  token_id >= vocab -> MMRS_ERR_ARG;
 * a non-finite result -> device status MMRS_ERR_NONFINITE. */
MMRS_API int mmrs_token_logprob(const float *logits, int vocab, int token_id, float *out, void *workspace,
                                size_t workspace_bytes, mmrs_stream_t stream);

/* ---- verification of drafted tokens ------------------------------------------------------ */

/* Sequences, logits rows and rows per sequence a call takes. */
#define MMRS_VERIFY_MAX_SEQS 1024
#define MMRS_VERIFY_MAX_ROWS 65536
#define MMRS_VERIFY_MAX_Q 64

/* Workspace bytes of mmrs_verify_drafts (0: arguments out of range).  Caller-owned, 256-byte
 * aligned, zero before first use; one workspace serves one stream at a time and calls of any size
 * up to its own. */
MMRS_API size_t mmrs_verify_workspace_bytes(int num_seqs, int total_rows);

/* Outcome of the last completed call on a workspace (synchronous read): MMRS_OK, or
 * MMRS_ERR_NONFINITE when some sequence's next token could not be chosen (its place holds -1). */
MMRS_API int mmrs_verify_workspace_status(const void *workspace);

/* No counterpart in the reference (it decodes one token at a time, src/sampling.rs:84-150).
 * Sequence b has the logits rows cu_rows[b] .. cu_rows[b + 1] - 1 of logits [total_rows][vocab]
 * (logits_type MMRS_TYPE_F32, _F16 or _BF16 of minimax_paged.h): the target's rows after its last
 * accepted token and after each of its d = rows - 1 drafted tokens.  Draft i of it, element
 * cu_rows[b] - b + i of draft_tokens and uniforms and row of draft_probs [drafts][vocab] (the draft
 * model's probabilities; null: the draft had probability 1), is judged by row i:
 *   temperature[b] == 0: it stands when it is the row's argmax (first index of the largest);
 *   otherwise, with p = softmax(logits / temperature[b]), when u * q(draft) < p(draft).
 * The drafts before the first that falls are emitted, then one more token: at temperature 0 the
 * argmax of the next row; else the argmax over the vocabulary (first index on ties) of r / noise[b],
 * noise [num_seqs][vocab] exponential random numbers, which draws from r: p of the last row when
 * all drafts stood, max(p - q, 0) of the row where one fell (p itself where that is nowhere
 * positive; with draft_probs null, p without the draft).
 * tokens int32 [num_seqs][max_q] = the emitted tokens, then -1; accepted int32 [num_seqs] = drafts
 * that stood; logprobs f32 [num_seqs][max_q] (or null) = ln softmax(logits / T) of the emitted tokens
 * in their rows (T = temperature, 1 where that is 0), then 0.  temperature f32 [num_seqs], or null: 1.
 * Logits of -infinity are masked tokens.  A draft judged by a row that holds NaN or +infinity, or
 * nothing but -infinity, falls; a next token that such a row should give is -1 (device status
 * MMRS_ERR_NONFINITE).  Sequences without rows come last and emit nothing.  max_q bounds the rows of a
 * sequence; total_rows bounds cu_rows. */
MMRS_API int mmrs_verify_drafts(const void *logits, int logits_type, int vocab, const int32_t *cu_rows, int num_seqs,
                                int total_rows, int max_q, const int32_t *draft_tokens, const float *draft_probs,
                                const float *uniforms, const float *noise, const float *temperature, int32_t *tokens,
                                int32_t *accepted, float *logprobs, void *workspace, size_t workspace_bytes,
                                mmrs_stream_t stream);

/* The same with the number of drafts: draft_tokens and uniforms have num_drafts elements, draft_probs
 * num_drafts rows, and nothing past them is read.  A draft that would lie there falls, and the next
 * token is drawn from p of its row.  (mmrs_verify_drafts takes arrays that hold a draft for every
 * row but each sequence's last; without them no draft stands.) */
MMRS_API int mmrs_verify_drafts_n(const void *logits, int logits_type, int vocab, const int32_t *cu_rows, int num_seqs,
                                  int total_rows, int max_q, const int32_t *draft_tokens, const float *draft_probs,
                                  const float *uniforms, int num_drafts, const float *noise, const float *temperature,
                                  int32_t *tokens, int32_t *accepted, float *logprobs, void *workspace,
                                  size_t workspace_bytes, mmrs_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* MINIMAX_SAMPLE_H */
