// Verification of drafted tokens against the target's probabilities (mmrs_verify_drafts).
//
// With c = log2(e) / T a row's probabilities are 2^(c (l - max)) / sum, and the next token is the argmax
// of r / e over the vocabulary (r: p, or what p has over q; e exponential: the first arrival of a race
// in which token i runs at rate r_i).  Both need every logit of a row once; nothing else is long, so
// the kernels are bound by HBM, or by the latency of two dependent passes where there are few rows.
//   verify_rows_kernel    (row, chunk): one read of the chunk leaves its maximum, its sum of
//                         exponentials and, for greedy rows, its argmax; a sequence's last block to
//                         finish joins its rows' chunks (a few hundred bytes) and judges the drafts;
//   verify_choose_kernel  (chunk, sequence): the race over a chunk of the row that gives the next token;
//                         the sequence's last block to finish joins the chunks' winners.  It starts
//                         while the first kernel drains, with its noise on the way.
// A block reads 64 bytes a thread at once and keeps them in registers: 8192 f32 or 16384 16-bit tokens
// (8192 of 16 bits: 33 ragged sequences 39 us instead of 37, 320 rows of f16 86 instead of 80; that the largest
// of 16-bit logits is found two at a time makes that 76).  A row is cut into the number of chunks whose rounds of
// resident blocks are the shortest.
// Measured (200064 tokens, with the draft model's probabilities unless said): 5 rows of f32 12.8 us in a
// captured graph (two launches and their dependent reads; the bytes alone would take 0.9); 320 rows of
// 64 sequences 74 us (362 MB, 4.9 TB/s, 0.74 of a plain copy's); 33 sequences of 1 to 8 bf16 rows without
// probabilities 37 us (floor 12: rounds of blocks that wait for their own reads).
#include <cuda_runtime.h>
#include <math.h>

#include <type_traits>

#include "../../include/minimax_sample.h"
#include "paged.cuh"
#include "tma.cuh"

namespace mmrs {
namespace {

constexpr int kVfThreads = 512;
constexpr int kVfWarps = kVfThreads / 32;
constexpr int kVfGroups = 4;                               // 16-byte reads that a thread holds
constexpr int kVfBlock = kVfThreads * kVfGroups * 4;       // f32 tokens a block reads at once
constexpr int kVfChunks = 32;                              // chunks of a row, at most
constexpr float kVfLog2e = 1.4426950408889634f;

struct VfPart {
    float top, sum;           // maximum of the logits and sum of 2^(c (l - top)); NaN: a logit was
    unsigned long long best;  // lm_key of the largest logit (greedy rows)
};
struct VfSeq {
    unsigned long long best[kVfChunks];  // lm_key of the chunks' winners, 0: none
    uint32_t rows_done, count;           // blocks done of either kernel, zero between calls
    int stood;                           // drafts that stand
    float top, sum;                      // of the row that gives the next token
    int greedy_next;                     // its argmax
};

struct VfParams {
    const void *logits;
    int vocab, num_seqs, total_rows, max_q;
    int num_drafts;               // elements of draft and u, rows of q
    int chunks, chunk;            // rows kernel: chunks of a row, tokens of a chunk
    int race_chunks, race_chunk;  // choose kernel
    const int32_t *cu, *draft;
    const float *q, *u, *noise, *temperature;
    int32_t *tokens, *accepted;
    float *logprobs;
    VfPart *parts;  // [row][chunk]
    VfSeq *seqs;
    uint32_t *status;
};

__device__ __forceinline__ float vf_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Four elements at i (a multiple of 4) of a row of n: one read where the row is aligned for it.
template <typename T>
__device__ __forceinline__ void vf_load4(const T *row, int i, int n, float fill, float (&x)[4]) {
    if (i + 4 <= n && ((uintptr_t)row & (4 * sizeof(T) - 1)) == 0) {
        pg_load4(row + i, x);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = i + k < n ? pg_to_float(row[i + k]) : fill;
    }
}
// 16 bytes at i (a multiple of their number of elements) of a row of n, as they are; -infinity past n.
template <typename T>
__device__ __forceinline__ uint4 vf_load16(const T *row, int i, int n) {
    constexpr int kN = 16 / sizeof(T);
    if (i + kN <= n && ((uintptr_t)(row + i) & 15) == 0) return *reinterpret_cast<const uint4 *>(row + i);
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 4) {
            w[k] = i + k < n ? reinterpret_cast<const uint32_t *>(row)[i + k] : 0xff800000u;
        } else {
            constexpr uint32_t kNone = __is_same(T, __half) ? 0xfc00u : 0xff80u;
            const uint16_t *r = reinterpret_cast<const uint16_t *>(row);
            w[k] = (i + 2 * k < n ? r[i + 2 * k] : kNone) | (i + 2 * k + 1 < n ? r[i + 2 * k + 1] : kNone) << 16;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// The elements of a word: one, or two.
__device__ __forceinline__ void vf_split(uint32_t w, float (&x)[1], const float *) { x[0] = __uint_as_float(w); }
__device__ __forceinline__ void vf_split(uint32_t w, float (&x)[2], const __half *) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    x[0] = f.x, x[1] = f.y;
}
__device__ __forceinline__ void vf_split(uint32_t w, float (&x)[2], const __nv_bfloat16 *) {
    x[0] = __uint_as_float(w << 16), x[1] = __uint_as_float(w & 0xffff0000u);
}
// The largest element of the words (NaN aside).
template <int kN>
__device__ __forceinline__ float vf_top(const uint32_t (&x)[kN], const float *) {
    float top = __uint_as_float(x[0]);
#pragma unroll
    for (int j = 1; j < kN; ++j) top = fmaxf(top, __uint_as_float(x[j]));
    return fmaxf(top, -INFINITY);
}
template <int kN, typename T>
__device__ __forceinline__ float vf_top(const uint32_t (&x)[kN], const T *t) {
    using T2 = std::conditional_t<__is_same(T, __half), __half2, __nv_bfloat162>;
    T2 top = *reinterpret_cast<const T2 *>(&x[0]);
#pragma unroll
    for (int j = 1; j < kN; ++j) top = __hmax2(top, *reinterpret_cast<const T2 *>(&x[j]));
    float e[2];
    vf_split(*reinterpret_cast<const uint32_t *>(&top), e, t);
    return fmaxf(fmaxf(e[0], e[1]), -INFINITY);
}
// (m, s) of the warp's parts: one rescaling each, then plain sums.
__device__ __forceinline__ void vf_join_warp(float &m, float &s, float c) {
    const float top = warp_max_butterfly(m);
    s = warp_sum_butterfly(s * vf_exp2((m - (top == -INFINITY ? 0.0f : top)) * c));
    m = top;
}
// (m, s) of two parts of a sum of exponentials with maxima m; -inf with sum 0 is nothing.
__device__ __forceinline__ void vf_join(float &m, float &s, float m2, float s2, float c) {
    const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.0f : top;
    s = s * vf_exp2((m - base) * c) + s2 * vf_exp2((m2 - base) * c);
    m = top;
}
__device__ __forceinline__ float vf_temperature(const VfParams &p, int s) { return p.temperature ? p.temperature[s] : 1.0f; }
__device__ __forceinline__ int vf_index(unsigned long long key) { return (int)(0xFFFFFFFFu - (uint32_t)key); }

// The whole row's maximum, sum and argmax (one warp; lanes hold chunks).
__device__ __forceinline__ VfPart vf_row(const VfParams &p, int row, int lane, float c) {
    VfPart r{-INFINITY, 0.0f, 0};
    if (lane < p.chunks) {
        const VfPart *part = p.parts + (long)row * kVfChunks + lane;
        r.top = __ldcg(&part->top), r.sum = __ldcg(&part->sum), r.best = __ldcg(&part->best);
    }
    vf_join_warp(r.top, r.sum, c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r.best = max(r.best, __shfl_xor_sync(0xffffffffu, r.best, o));
    return r;
}

// The sequence's drafts judged (whole block): one warp a row.
template <typename T>
__device__ __forceinline__ void vf_judge(const VfParams &p, int s, int row0, int rows, float t0) {
    __shared__ VfPart s_row[MMRS_VERIFY_MAX_Q];
    __shared__ bool s_stands[MMRS_VERIFY_MAX_Q];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool greedy = t0 == 0.0f;
    const float c = greedy ? kVfLog2e : kVfLog2e / t0;
    for (int r = warp; r < rows; r += kVfWarps) {
        const int row = row0 + r, at = row - s;
        float l = 0.0f, q = 1.0f, u = 0.0f;
        int tok = -1;
        if (r < rows - 1 && at >= 0 && at < p.num_drafts) {  // (no draft there: it falls)
            tok = p.draft[at], u = p.u[at];
            if (tok >= 0 && tok < p.vocab) {
                l = pg_to_float(static_cast<const T *>(p.logits)[(long)row * p.vocab + tok]);
                if (p.q) q = p.q[(long)at * p.vocab + tok];
            }
        }
        const VfPart part = vf_row(p, row, lane, c);
        if (lane == 0) {
            s_row[r] = part;
            const float pr = vf_exp2((l - part.top) * c) / part.sum;
            s_stands[r] = part.sum > 0.0f && tok >= 0 && tok < p.vocab &&
                          (greedy ? vf_index(part.best) == tok : u * q < pr);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int n = 0;
        while (n < rows - 1 && s_stands[n]) ++n;
        VfSeq *seq = p.seqs + s;
        seq->stood = n, seq->top = s_row[n].top, seq->sum = s_row[n].sum;
        seq->greedy_next = vf_index(s_row[n].best);
        seq->rows_done = 0;
    }
}

template <typename T>
__global__ void __launch_bounds__(kVfThreads, sizeof(T) == 4 ? 4 : 3) verify_rows_kernel(const VfParams p) {
    __shared__ float s_m[kVfWarps], s_s[kVfWarps];
    __shared__ unsigned long long s_b[kVfWarps];
    __shared__ int s_last;
    launch_dependents();
    const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (row == 0 && blockIdx.y == 0 && threadIdx.x == 0) *p.status = MMRS_OK;
    if (row >= p.total_rows) return;
    const T *l = static_cast<const T *>(p.logits) + (long)row * p.vocab;
    const int c0 = blockIdx.y * p.chunk, c1 = min(c0 + p.chunk, p.vocab);
    constexpr int kN = 16 / sizeof(T), kW = 4 / sizeof(T);  // elements of a read and of a word of it
    uint32_t x[4 * kVfGroups];
    auto load = [&](int i0) {
#pragma unroll
        for (int j = 0; j < kVfGroups; ++j) {
            const uint4 r = vf_load16(l, i0 + (j * kVfThreads + (int)threadIdx.x) * kN, c1);
            x[4 * j] = r.x, x[4 * j + 1] = r.y, x[4 * j + 2] = r.z, x[4 * j + 3] = r.w;
        }
    };
    load(c0);  // on the way while the row's sequence is looked up
    int s = 0;
    for (int s0 = 0; s0 < p.num_seqs; s0 += 32)
        s += __popc(__ballot_sync(0xffffffffu, s0 + lane < p.num_seqs && p.cu[s0 + lane + 1] <= row));
    if (s >= p.num_seqs) return;  // a row past the last sequence's
    const float t = vf_temperature(p, s);
    const bool greedy = t == 0.0f;
    const float c = greedy ? kVfLog2e : kVfLog2e / t;
    float m = -INFINITY, sum = 0.0f, best = -INFINITY;
    int at = -1;
    for (int i0 = c0;;) {
        const float top = vf_top(x, (const T *)nullptr);
        if (greedy) {
#pragma unroll
            for (int j = 0; j < 4 * kVfGroups; ++j) {
                float e[kW];
                vf_split(x[j], e, (const T *)nullptr);
#pragma unroll
                for (int k = 0; k < kW; ++k)
                    if (e[k] > best)
                        best = e[k], at = i0 + ((j / 4) * kVfThreads + (int)threadIdx.x) * kN + (j % 4) * kW + k;
            }
        }
        // (the words are taken apart a second time: twice as many floats would not stay in registers)
#pragma unroll
        for (int j = 0; j < 4 * kVfGroups; ++j)
            if constexpr (kW == 2) asm volatile("" : "+r"(x[j]));
        const float base = top == -INFINITY ? 0.0f : top;
        float part = 0.0f;
#pragma unroll
        for (int j = 0; j < 4 * kVfGroups; ++j) {
            float e[kW];
            vf_split(x[j], e, (const T *)nullptr);
#pragma unroll
            for (int k = 0; k < kW; ++k) part += vf_exp2((e[k] - base) * c);  // an infinity leaves NaN here
        }
        vf_join(m, sum, top, part, c);
        i0 += kVfThreads * kVfGroups * kN;
        if (i0 >= c1) break;
        load(i0);
    }
    unsigned long long key = at >= 0 ? lm_key(best, at) : 0;
    vf_join_warp(m, sum, c);
    if (greedy)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
    if (lane == 0) s_m[warp] = m, s_s[warp] = sum, s_b[warp] = key;
    __syncthreads();
    if (warp == 0) {
        m = lane < kVfWarps ? s_m[lane] : -INFINITY, sum = lane < kVfWarps ? s_s[lane] : 0.0f;
        key = lane < kVfWarps ? s_b[lane] : 0;
        vf_join_warp(m, sum, c);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
        if (lane == 0) {
            p.parts[(long)row * kVfChunks + blockIdx.y] = VfPart{m, sum, key};
            const int row0 = max(p.cu[s], 0), rows = min(min(p.cu[s + 1], p.total_rows) - row0, p.max_q);
            __threadfence();
            // (rows past max_q are not counted)
            s_last = row < row0 + rows && atomicAdd(&p.seqs[s].rows_done, 1u) + 1 == (uint32_t)rows * p.chunks;
            __threadfence();
        }
    }
    __syncthreads();
    if (!s_last) return;
    const int row0 = max(p.cu[s], 0);
    vf_judge<T>(p, s, row0, min(min(p.cu[s + 1], p.total_rows) - row0, p.max_q), t);
}

template <typename T>
__global__ void __launch_bounds__(kVfThreads, 2) verify_choose_kernel(const VfParams p) {
    __shared__ unsigned long long s_b[kVfWarps];
    __shared__ int s_last;
    const int s = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row0 = max(p.cu[s], 0), rows = min(min(p.cu[s + 1], p.total_rows) - row0, p.max_q);
    const float t0 = vf_temperature(p, s), t = t0 == 0.0f ? 1.0f : t0, c = kVfLog2e / t;
    const bool greedy = t0 == 0.0f;
    const int c0 = blockIdx.x * p.race_chunk, c1 = min(c0 + p.race_chunk, p.vocab);
    const float *noise = p.noise + (long)s * p.vocab;
    float e[kVfGroups][4];
    if (!greedy && rows > 0)
#pragma unroll
        for (int j = 0; j < kVfGroups; ++j) vf_load4(noise, c0 + (j * kVfThreads + threadIdx.x) * 4, c1, 1.0f, e[j]);
    grid_dependency_wait();
    int32_t *tokens = p.tokens + (long)s * p.max_q;
    float *logprobs = p.logprobs ? p.logprobs + (long)s * p.max_q : nullptr;
    const T *logits = static_cast<const T *>(p.logits);
    VfSeq *seq = p.seqs + s;
    const int n = rows > 0 ? min(max(__ldcg(&seq->stood), 0), rows - 1) : 0;  // (a row of the sequence, whatever is there)
    const float top = __ldcg(&seq->top), sum = __ldcg(&seq->sum);
    const int row = row0 + n, at = row - s;
    const bool usable = rows > 0 && sum > 0.0f, fell = n < rows - 1 && at >= 0 && at < p.num_drafts;
    const T *l = logits + (long)row * p.vocab;
    const float *q = fell && p.q ? p.q + (long)at * p.vocab : nullptr;
    const int gone = fell && !p.q ? p.draft[at] : -1;
    // the race over tokens [i0, i1) of the row; `own`: against the draft's probabilities
    auto race = [&](int i0, int i1, bool first, bool own) {
        const float inv = 1.0f / sum;
        float best = 0.0f;
        int win = -1;
        for (; i0 < i1; i0 += kVfBlock, first = false) {
            float x[kVfGroups][4], y[kVfGroups][4];
#pragma unroll
            for (int j = 0; j < kVfGroups; ++j) {
                const int i = i0 + (j * kVfThreads + threadIdx.x) * 4;
                vf_load4(l, i, i1, -INFINITY, x[j]);
                if (own && q) vf_load4(q, i, i1, 0.0f, y[j]);
                if (!first) vf_load4(noise, i, i1, 1.0f, e[j]);
            }
#pragma unroll
            for (int j = 0; j < kVfGroups; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i = i0 + (j * kVfThreads + (int)threadIdx.x) * 4 + k;
                    float r = vf_exp2((x[j][k] - top) * c) * inv;
                    if (own) r = q ? r - y[j][k] : i == gone ? 0.0f : r;
                    const float v = __fdividef(r, e[j][k]);
                    if (r > 0.0f && v > best) best = v, win = i;  // indices rise: the first of equals stays
                }
        }
        unsigned long long key = win >= 0 ? lm_key(best, win) : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
        __syncthreads();
        if (lane == 0) s_b[warp] = key;
        __syncthreads();
        for (int w = 0; w < kVfWarps; ++w) key = max(key, s_b[w]);
        return key;
    };
    if (usable && !greedy) {
        const unsigned long long key = race(c0, c1, true, true);
        if (threadIdx.x == 0) {
            __stcg(&seq->best[blockIdx.x], key);
            __threadfence();
            s_last = atomicAdd(&seq->count, 1u) + 1 == gridDim.x;
            __threadfence();
        }
        __syncthreads();
        if (!s_last) return;
    } else if (blockIdx.x > 0) {
        return;
    }
    // one block a sequence from here on
    int next = -1;
    if (usable && greedy) next = __ldcg(&seq->greedy_next);
    if (usable && !greedy) {
        unsigned long long key = 0;
        for (int i = 0; i < p.race_chunks; ++i) key = max(key, __ldcg(&seq->best[i]));
        if (!key) key = race(0, p.vocab, false, false);  // nothing was left of p: the target's own race
        if (key) next = vf_index(key);
        if (threadIdx.x == 0) seq->count = 0;
    }
    if (threadIdx.x == 0) {
        p.accepted[s] = n;
        if (rows > 0 && next < 0) atomicExch(p.status, (uint32_t)MMRS_ERR_NONFINITE);
    }
    for (int i = warp; i < p.max_q; i += kVfWarps) {
        const int tok = rows <= 0 || i > n ? -1 : i < n ? p.draft[row0 + i - s] : next;
        float lp = 0.0f;
        if (logprobs && tok >= 0) {
            const VfPart part = vf_row(p, row0 + i, lane, c);
            lp = (pg_to_float(logits[(long)(row0 + i) * p.vocab + tok]) - part.top) / t - logf(part.sum);
        }
        if (lane == 0) {
            tokens[i] = tok;
            if (logprobs) logprobs[i] = lp;
        }
    }
}

// Workspace: a status word, the sequences' records, the rows' parts.  The records' counters are zero from one
// call to the next, so they lie where no call's size moves them (room for the most sequences, 287 KB): else a
// call of few sequences would write its parts over the records that a larger one finds.
constexpr size_t kVfSeqsAt = 256;
constexpr size_t kVfPartsAt = kVfSeqsAt + (sizeof(VfSeq) * MMRS_VERIFY_MAX_SEQS + 255) / 256 * 256;
size_t vf_workspace_bytes(int num_seqs, int total_rows) {
    if (num_seqs < 0 || num_seqs > MMRS_VERIFY_MAX_SEQS || total_rows < 0 || total_rows > MMRS_VERIFY_MAX_ROWS) return 0;
    return kVfPartsAt + sizeof(VfPart) * kVfChunks * (size_t)total_rows;
}

template <typename T>
int vf_launch(const VfParams &p, cudaStream_t s) {
    // (at least one block of the first kernel: it resets the status)
    verify_rows_kernel<T><<<dim3(p.total_rows > 0 ? p.total_rows : 1, p.chunks), kVfThreads, 0, s>>>(p);
    if (cudaGetLastError() != cudaSuccess) return MMRS_ERR_LAUNCH;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.race_chunks, p.num_seqs);
    cfg.blockDim = dim3(kVfThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, verify_choose_kernel<T>, p) == cudaSuccess ? MMRS_OK : MMRS_ERR_LAUNCH;
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

extern "C" int mmrs_verify_drafts_n(const void *logits, int logits_type, int vocab, const int32_t *cu_rows, int num_seqs,
                                    int total_rows, int max_q, const int32_t *draft_tokens, const float *draft_probs,
                                    const float *uniforms, int num_drafts, const float *noise, const float *temperature,
                                    int32_t *tokens, int32_t *accepted, float *logprobs, void *workspace,
                                    size_t workspace_bytes, mmrs_stream_t stream) {
    if (logits_type < MMRS_TYPE_F32 || logits_type > MMRS_TYPE_BF16) return MMRS_ERR_UNSUPPORTED;
    if (vocab < 1 || vocab > MMRS_SAMPLE_MAX_VOCAB || num_seqs < 0 || num_seqs > MMRS_VERIFY_MAX_SEQS ||
        total_rows < 0 || total_rows > MMRS_VERIFY_MAX_ROWS || max_q < 1 || max_q > MMRS_VERIFY_MAX_Q || num_drafts < 0)
        return MMRS_ERR_ARG;
    if (num_seqs == 0) return MMRS_OK;
    if (!cu_rows || !tokens || !accepted) return MMRS_ERR_ARG;
    if (total_rows && (!logits || !noise)) return MMRS_ERR_ARG;
    if (num_drafts && (!draft_tokens || !uniforms)) return MMRS_ERR_ARG;
    if (!workspace || ((uintptr_t)workspace & 255u) || workspace_bytes < vf_workspace_bytes(num_seqs, total_rows))
        return MMRS_ERR_ARG;
    VfParams p = {};
    p.logits = logits;
    p.vocab = vocab, p.num_seqs = num_seqs, p.total_rows = total_rows, p.max_q = max_q;
    p.num_drafts = num_drafts;
    p.cu = cu_rows, p.draft = draft_tokens;
    p.q = draft_probs, p.u = uniforms, p.noise = noise, p.temperature = temperature;
    p.tokens = tokens, p.accepted = accepted, p.logprobs = logprobs;
    // chunks of a row: of all numbers of them the one whose rounds of resident blocks (a block's beginning
    // and end count as two reads of a block) are the shortest in all, fewer chunks first
    auto chunk_of = [&](long rows, int resident, int block) {
        const int most = (vocab + block - 1) / block;
        long best = -1;
        int chunk = 0;
        for (int n = 1; n <= kVfChunks && n <= most; ++n) {
            const int reads = (most + n - 1) / n;
            const long rounds = (rows * ((most + reads - 1) / reads) + 148L * resident - 1) / (148L * resident);
            const long cost = rounds * (reads + 2);
            if (best < 0 || cost < best) best = cost, chunk = reads * block;
        }
        return chunk;
    };
    p.chunk = logits_type == MMRS_TYPE_F32 ? chunk_of(total_rows, 4, kVfBlock) : chunk_of(total_rows, 3, 2 * kVfBlock);
    p.race_chunk = chunk_of(num_seqs, 2, kVfBlock);
    p.chunks = (vocab + p.chunk - 1) / p.chunk;
    p.race_chunks = (vocab + p.race_chunk - 1) / p.race_chunk;
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    p.status = reinterpret_cast<uint32_t *>(ws);
    p.seqs = reinterpret_cast<VfSeq *>(ws + kVfSeqsAt);
    p.parts = reinterpret_cast<VfPart *>(ws + kVfPartsAt);
    cudaStream_t s = (cudaStream_t)stream;
    if (logits_type == MMRS_TYPE_F32) return vf_launch<float>(p, s);
    return logits_type == MMRS_TYPE_F16 ? vf_launch<__half>(p, s) : vf_launch<__nv_bfloat16>(p, s);
}

extern "C" int mmrs_verify_drafts(const void *logits, int logits_type, int vocab, const int32_t *cu_rows, int num_seqs,
                                  int total_rows, int max_q, const int32_t *draft_tokens, const float *draft_probs,
                                  const float *uniforms, const float *noise, const float *temperature, int32_t *tokens,
                                  int32_t *accepted, float *logprobs, void *workspace, size_t workspace_bytes,
                                  mmrs_stream_t stream) {
    // How many sequences have rows is on the device: more rows than sequences bring drafts for certain; without
    // the arrays there are none, with them as many as the rows ask for.
    const bool given = draft_tokens && uniforms;
    if (total_rows > num_seqs && num_seqs > 0 && !given) return MMRS_ERR_ARG;
    return mmrs_verify_drafts_n(logits, logits_type, vocab, cu_rows, num_seqs, total_rows, max_q, draft_tokens, draft_probs,
                                uniforms, given && total_rows > 0 ? total_rows : 0, noise, temperature, tokens, accepted,
                                logprobs, workspace, workspace_bytes, stream);
}
