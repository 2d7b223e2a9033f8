// Pieces shared by the two paged attention kernels: arguments, the work list over sequences and
// KV heads, the visible positions of a sequence, and the merge of partial results.
#pragma once

#include <math.h>

#include "paged.cuh"
#include "tma.cuh"

namespace mmrs {

constexpr int kPaMaxSeqs = MMRS_PAGED_MAX_SEQS;
constexpr int kPaDecodeRows = 32;  // rows of an item of the decode kernel, at most
// Rows of a KV head up to which a sequence is the decode kernel's: 64 sequences (300000 positions, 8
// heads) take it 242 us with 30 rows, 362 with 48, 462 with 54, 695 with 96, and the prompt kernel 313 to
// 330 with any number from 30 to 96; 4 sequences 32 us with 30 rows, 36 with 48, 44 with 54, 58 with 96, and 45 to 51.
constexpr int kPaFewRows = 48;
constexpr float kPaLog2e = 1.4426950408889634f;
constexpr float kPaLn2 = 0.6931471805599453f;
constexpr uint64_t kPaTimeoutNs = 2000000000ull;

struct PaParams {
    MmrsPagedCache c;
    MmrsPagedBatch b;
    const void *q;
    void *out;
    float *lse;
    long q_stride;
    int query_heads, group, window, sinks;
    int few_rows;  // sequences of at most this many rows a KV head are the decode kernel's, others the prompt kernel's
    bool mixed;    // both kernels run
    float scale_log2;     // scale * log2(e)
    uint32_t *status;     // workspace: status word
    uint32_t *counters;   // workspace: one per CTA (for the item it begins and others end), zero between calls
    float *partials;      // workspace: two slots per CTA, for the items it shares with CTAs before and after it
};

// The positions that some new token of a sequence sees, in steps of kStep: the steps [0, ns) of
// the first tokens that stay visible, then [first, ns + ... ) up to the length.
template <int kStep>
struct PaSpan {
    int ns, first, n;
    __device__ __forceinline__ int step(int i) const { return i < ns ? i : i - ns + first; }
};
// `lo`, `hi`: the positions of the first and last of the rows concerned (hi < the sequence's length).
template <int kStep>
__device__ __forceinline__ PaSpan<kStep> pa_span(int lo, int hi, int window, int sinks) {
    PaSpan<kStep> s;
    const int end = hi / kStep + 1;  // hi >= -1
    s.ns = 0, s.first = 0;
    if (window > 0) {
        const int from = lo - window + 1;
        s.ns = sinks > 0 ? min((min(sinks, hi + 1) + kStep - 1) / kStep, end) : 0;
        s.first = from > 0 ? max(from / kStep, s.ns) : s.ns;
    }
    s.n = hi < 0 ? 0 : s.ns + max(0, end - s.first);
    return s;
}
__device__ __forceinline__ bool pa_sees(int j, int pos, int window, int sinks) {
    return j <= pos && (window <= 0 || pos - j < window || j < sinks);
}

// 2^x; -inf gives 0.
__device__ __forceinline__ float pa_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A tile of a 2-D byte matrix into shared memory.
__device__ __forceinline__ void pa_tma_2d(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}

// Rows of 128 codes, read `rows` at a time with the 128-byte swizzle (16-byte chunk index xor row & 7).
int pa_make_map(CUtensorMap *map, const void *codes, const MmrsPagedCache &c, int rows);

int pa_sm_count();

// Kernels' launchers.
int pa_launch_decode(const PaParams &p, const CUtensorMap &k, const CUtensorMap &v, int type, cudaStream_t s);
int pa_launch_prompt(const PaParams &p, int type, cudaStream_t s);

}  // namespace mmrs
