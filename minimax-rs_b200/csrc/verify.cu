// Verification of drafted tokens against the target's probabilities (mmrs_verify_drafts).
//
// rows_kernel: one CTA per logits row reads it once and leaves its maximum, sum of exp(x - max)
// and argmax (x = logits / T).  choose_kernel: one CTA per sequence walks its rows' judgements
// (a draft stands when u q < p), then runs the exponential race argmax r / e over the vocabulary
// for the row that gives the next token.
#include <cuda_runtime.h>
#include <math.h>

#include "../../include/minimax_sample.h"
#include "paged.cuh"

namespace mmrs {
namespace {

constexpr int kVfThreads = 512;
constexpr int kVfWarps = kVfThreads / 32;

struct VfRow {
    float top, sum;            // maximum of x and sum of exp(x - top); sum 0: no usable row
    unsigned long long best;   // lm_key of the largest logit
};

struct VfParams {
    const void *logits;
    int vocab, num_seqs, total_rows, max_q;
    const int32_t *cu, *draft;
    const float *q, *u, *noise, *temperature;
    int32_t *tokens, *accepted;
    float *logprobs;
    VfRow *rows;
    uint32_t *status;
};

template <typename T>
__device__ __forceinline__ float vf_logit(const void *p, long i) {
    return pg_to_float(static_cast<const T *>(p)[i]);
}

template <typename T>
__global__ void __launch_bounds__(kVfThreads) verify_rows_kernel(const VfParams p) {
    __shared__ float s_m[kVfWarps], s_s[kVfWarps];
    __shared__ unsigned long long s_b[kVfWarps];
    const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = 0;
    for (int s0 = 0; s0 < p.num_seqs; s0 += 32)
        s += __popc(__ballot_sync(0xffffffffu, s0 + lane < p.num_seqs && p.cu[s0 + lane + 1] <= row));
    float t = p.temperature && s < p.num_seqs ? p.temperature[s] : 1.0f;
    if (t == 0.0f) t = 1.0f;
    float m = -INFINITY, sum = 0.0f;
    unsigned long long best = 0;
    bool bad = false;
    for (int i = threadIdx.x; i < p.vocab; i += kVfThreads) {
        const float l = vf_logit<T>(p.logits, (long)row * p.vocab + i), x = l / t;
        bad = bad || !(l < INFINITY);
        const unsigned long long key = lm_key(l, i);
        best = key > best ? key : best;
        if (x > m) {
            sum = sum * expf(m - x) + 1.0f;
            m = x;
        } else if (x != -INFINITY) {
            sum += expf(x - m);
        }
    }
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, sum, o);
        const float mm = fmaxf(m, m2);
        sum = mm == -INFINITY ? 0.0f : sum * expf(m - mm) + s2 * expf(m2 - mm);
        m = mm;
        const unsigned long long b2 = __shfl_xor_sync(0xffffffffu, best, o);
        best = b2 > best ? b2 : best;
    }
    bad = __syncthreads_or(bad);
    if (lane == 0) s_m[warp] = m, s_s[warp] = sum, s_b[warp] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kVfWarps; ++w) {
            const float mm = fmaxf(m, s_m[w]);
            sum = mm == -INFINITY ? 0.0f : sum * expf(m - mm) + s_s[w] * expf(s_m[w] - mm);
            m = mm;
            best = s_b[w] > best ? s_b[w] : best;
        }
        p.rows[row].top = m;
        p.rows[row].sum = bad ? 0.0f : sum;
        p.rows[row].best = best;
    }
}

template <typename T>
__global__ void __launch_bounds__(kVfThreads) verify_choose_kernel(const VfParams p) {
    __shared__ unsigned long long s_b[kVfWarps];
    const int s = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row0 = max(p.cu[s], 0), rows = min(min(p.cu[s + 1], p.total_rows) - row0, p.max_q);
    const float t0 = p.temperature ? p.temperature[s] : 1.0f, t = t0 == 0.0f ? 1.0f : t0;
    int32_t *tokens = p.tokens + (long)s * p.max_q;
    float *logprobs = p.logprobs ? p.logprobs + (long)s * p.max_q : nullptr;
    for (int i = threadIdx.x; i < p.max_q; i += kVfThreads) {
        tokens[i] = -1;
        if (logprobs) logprobs[i] = 0.0f;
    }
    if (rows <= 0) {
        if (threadIdx.x == 0) p.accepted[s] = 0;
        return;
    }
    __syncthreads();
    int n = 0;
    for (; n < rows - 1; ++n) {  // every thread judges alike
        const int row = row0 + n, at = row - s;
        if (at < 0) break;
        const int tok = p.draft[at];
        const VfRow r = p.rows[row];
        if (!(r.sum > 0.0f) || tok < 0 || tok >= p.vocab) break;
        const float x = vf_logit<T>(p.logits, (long)row * p.vocab + tok) / t;
        bool stands;
        if (t0 == 0.0f) {
            stands = tok == (int)(0xFFFFFFFFu - (uint32_t)r.best);
        } else {
            const float pr = expf(x - r.top) / r.sum, q = p.q ? p.q[(long)at * p.vocab + tok] : 1.0f;
            stands = p.u[at] * q < pr;
        }
        if (!stands) break;
        if (threadIdx.x == 0) {
            tokens[n] = tok;
            if (logprobs) logprobs[n] = (x - r.top) - logf(r.sum);
        }
    }
    const int row = row0 + n;
    const VfRow r = p.rows[row];
    int next = -1;
    if (r.sum > 0.0f && t0 == 0.0f) next = (int)(0xFFFFFFFFu - (uint32_t)r.best);
    if (r.sum > 0.0f && t0 != 0.0f) {
        const bool fell = n < rows - 1;
        unsigned long long best = 0, plain = 0;
        const int tok = fell && row >= s ? p.draft[row - s] : -1;
        const float *q = fell && p.q && row >= s ? p.q + (long)(row - s) * p.vocab : nullptr;
        for (int i = threadIdx.x; i < p.vocab; i += kVfThreads) {
            const float x = vf_logit<T>(p.logits, (long)row * p.vocab + i) / t;
            const float pr = expf(x - r.top) / r.sum;
            float rest = q ? fmaxf(pr - q[i], 0.0f) : fell && !p.q && i == tok ? 0.0f : pr;
            const float e = p.noise[(long)s * p.vocab + i];
            if (rest > 0.0f) best = max(best, lm_key(rest / e, i));
            if (pr > 0.0f) plain = max(plain, lm_key(pr / e, i));
        }
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        for (int o = 16; o > 0; o >>= 1) plain = max(plain, __shfl_xor_sync(0xffffffffu, plain, o));
        if (lane == 0) s_b[warp] = best;
        __syncthreads();
        for (int w = 0; w < kVfWarps; ++w) best = max(best, s_b[w]);
        __syncthreads();
        if (lane == 0) s_b[warp] = plain;
        __syncthreads();
        for (int w = 0; w < kVfWarps; ++w) plain = max(plain, s_b[w]);
        if (!best) best = plain;
        if (best) next = (int)(0xFFFFFFFFu - (uint32_t)best);
    }
    if (threadIdx.x == 0) {
        p.accepted[s] = n;
        tokens[n] = next;
        if (next < 0) atomicExch(p.status, (uint32_t)MMRS_ERR_NONFINITE);
        if (next >= 0 && logprobs)
            logprobs[n] = (vf_logit<T>(p.logits, (long)row * p.vocab + next) / t - r.top) - logf(r.sum);
    }
}

size_t vf_workspace_bytes(int num_seqs, int total_rows) {
    if (num_seqs < 0 || num_seqs > MMRS_VERIFY_MAX_SEQS || total_rows < 0 || total_rows > MMRS_VERIFY_MAX_ROWS) return 0;
    return 256 + sizeof(VfRow) * (size_t)total_rows;
}

template <typename T>
int vf_launch(const VfParams &p, cudaStream_t s) {
    if (cudaMemsetAsync(p.status, 0, sizeof(uint32_t), s) != cudaSuccess) return MMRS_ERR_LAUNCH;
    if (p.total_rows) verify_rows_kernel<T><<<p.total_rows, kVfThreads, 0, s>>>(p);
    verify_choose_kernel<T><<<p.num_seqs, kVfThreads, 0, s>>>(p);
    return cudaGetLastError() == cudaSuccess ? MMRS_OK : MMRS_ERR_LAUNCH;
}

}  // namespace
}  // namespace mmrs

using namespace mmrs;

extern "C" size_t mmrs_verify_workspace_bytes(int num_seqs, int total_rows) {
    return vf_workspace_bytes(num_seqs, total_rows);
}

extern "C" int mmrs_verify_workspace_status(const void *workspace) {
    if (!workspace) return MMRS_ERR_ARG;
    uint32_t st = 0;
    if (cudaMemcpy(&st, workspace, sizeof(st), cudaMemcpyDeviceToHost) != cudaSuccess) return MMRS_ERR_LAUNCH;
    return (int)st;
}

extern "C" int mmrs_verify_drafts(const void *logits, int logits_type, int vocab, const int32_t *cu_rows, int num_seqs,
                                  int total_rows, int max_q, const int32_t *draft_tokens, const float *draft_probs,
                                  const float *uniforms, const float *noise, const float *temperature, int32_t *tokens,
                                  int32_t *accepted, float *logprobs, void *workspace, size_t workspace_bytes,
                                  mmrs_stream_t stream) {
    if (logits_type < MMRS_TYPE_F32 || logits_type > MMRS_TYPE_BF16) return MMRS_ERR_UNSUPPORTED;
    if (vocab < 1 || vocab > MMRS_SAMPLE_MAX_VOCAB || num_seqs < 0 || num_seqs > MMRS_VERIFY_MAX_SEQS ||
        total_rows < 0 || total_rows > MMRS_VERIFY_MAX_ROWS || max_q < 1 || max_q > MMRS_VERIFY_MAX_Q)
        return MMRS_ERR_ARG;
    if (num_seqs == 0) return MMRS_OK;
    if (!cu_rows || !tokens || !accepted) return MMRS_ERR_ARG;
    if (total_rows && (!logits || !noise)) return MMRS_ERR_ARG;
    // a sequence may have no rows, so only more rows than sequences are known to bring drafts
    if (total_rows > num_seqs && (!draft_tokens || !uniforms)) return MMRS_ERR_ARG;
    if (!workspace || ((uintptr_t)workspace & 255u) || workspace_bytes < vf_workspace_bytes(num_seqs, total_rows))
        return MMRS_ERR_ARG;
    VfParams p = {};
    p.logits = logits;
    p.vocab = vocab, p.num_seqs = num_seqs, p.total_rows = total_rows, p.max_q = max_q;
    p.cu = cu_rows, p.draft = draft_tokens;
    p.q = draft_probs, p.u = uniforms, p.noise = noise, p.temperature = temperature;
    p.tokens = tokens, p.accepted = accepted, p.logprobs = logprobs;
    p.status = static_cast<uint32_t *>(workspace);
    p.rows = reinterpret_cast<VfRow *>(static_cast<uint8_t *>(workspace) + 256);
    cudaStream_t s = (cudaStream_t)stream;
    if (logits_type == MMRS_TYPE_F32) return vf_launch<float>(p, s);
    return logits_type == MMRS_TYPE_F16 ? vf_launch<__half>(p, s) : vf_launch<__nv_bfloat16>(p, s);
}
