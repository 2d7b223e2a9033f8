// Paged attention for few rows: single tokens and drafted tokens (at most kPaFewRows rows a KV head, in
// groups of up to 32, an item each; a kernel for 8, 16, 24 and 32 rows).
//
// Each K / V code is read once and used for all rows of its KV head, so the kernel is bound by HBM:
// 256 bytes a position and head.  The products run on mma.sync with the operands turned round, S^T =
// K Q^T and O^T += V^T P^T: 16 positions are the 16 rows of an instruction and eight
// query rows its columns, so that six query heads waste two columns of eight instead of ten rows
// of sixteen.  Which code goes to which contraction index is free as long as both operands agree,
// so a lane takes 32 consecutive codes of a key row (two 16-byte reads) and 16 of a value row, and
// turns them into f16 pairs in registers (e4m3 to f16 is exact).  P^T comes from S^T's accumulators
// by a transposing move of 8x8 tiles.
//
// The running maximum of a column moves only when a score passes it by more than 2^8 (P then still
// fits f16), found by one vote over the step's scores: the usual step neither reduces a maximum over
// lanes nor touches O.
//
// Value scales: P takes the ratio of its page's scale to the warp's reference, a power of two in f16.  The
// reference moves, and O with it, only for a page that has weight and lies above twice or below 1/64 of it.
// (A reference that went up only lost every value on pages 2^24 and more below the largest one met, and
// bits from 2^-14 on; the time is the same, 242 instead of 250 us for the drafts below.)
//
// Work: the steps of 32 positions of all sequences and KV heads form one list, of which every CTA
// (one per SM) takes an equal, contiguous part; a CTA's warps take its steps in turn, each
// with a ring of TMA copies of its own, its own running maximum and sum, and no barrier until the end
// of a (sequence, head).  Where that end lies in another CTA, the CTAs' partial results go through
// the workspace and the last to arrive joins them in order.
//
// Measured (48 + 8 heads): one token over 196608 positions 74 us (403 MB, 5.4 TB/s, 0.83 of a plain
// copy's; the same ring without the arithmetic takes 67); one token over 4096 positions 11.6 us call
// after call (a chain of latencies: launch, lookups, first tiles, joins); 64 sequences of 1001 to 8192
// positions and 5 drafted tokens (30 rows) 242 us (612 MB, 2.5 TB/s): eight warps of 255 registers, each
// with a chain of 128 products, 512 codes to turn and 32 exponentials a lane in a step, leave the
// issue slots two thirds empty and memory at 0.37.  Twelve warps of 168 registers, two a step: 475 us.
#include "paged_attend.cuh"

#include <algorithm>
#include <mutex>

namespace mmrs {
namespace {

constexpr int kPdStep = 32;                       // positions of a step: two groups of 16, each in one page
constexpr int kPdTile = kPdStep * kPgDim;         // bytes of its keys (or values)
constexpr float kPdLazy = 8.0f;                   // log2 of how far P may exceed 1
constexpr float kPdNone = -1e30f;                 // below every score
constexpr float kPdUnder = 1.0f / 64;             // how far a page's value scale may lie below the warp's reference
constexpr int kPdRowFloats = kPgDim + 4;          // a row of the merge buffer

constexpr int kPdWarps = 8;
constexpr int kPdThreads = 32 * kPdWarps;
constexpr int kPdStages = 2;
// What beginning and ending a (sequence, head) costs a block, in steps: the list is cut into equal
// parts with that much added to each item, else blocks over many short sequences end last (at 64
// sequences of 1000 to 8000 positions the last block took 1.4 times the average).
constexpr int kPdItemCost = 24;

template <int NT>
struct PdShared {
    uint8_t ring[kPdWarps][kPdStages][2][kPdTile];  // 1024-byte aligned tiles (swizzled)
    float o[kPdWarps / 2][8 * NT][kPdRowFloats];    // half the warps' sums
    uint32_t q[NT > 2 ? 8 : 1][4][32][2];           // NT = 3, 4: the queries' fragments
    float m[kPdWarps][32], l[kPdWarps][32];
    float4 meta[kPdWarps][kPdStages];               // k, v scale of the stage's two groups (k < 0: nothing there)
    uint64_t full[kPdWarps][kPdStages];
    int prefix[kPaMaxSeqs + 1];
    int scan[kPdWarps];
    int last;
};

__device__ __forceinline__ void pd_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pd_transpose(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint4 pd_lds(const uint8_t *tile, int row, int chunk) {
    return *reinterpret_cast<const uint4 *>(tile + row * kPgDim + ((chunk ^ (row & 7)) << 4));
}
// An item's piece in this CTA's part of the list: sequence b, KV head h, rows [row0, row0 + kRows) of
// the sequence's, steps [off, off + n) of the item's nb; the item's first step is unit `first` of the
// list, after its cost.
struct PdSeg {
    int b, h, row0, off, n, nb, first;
    PgSeq seq;
    PaSpan<kPdStep> span;
};

template <int NT, typename T>
struct PdKernel {
    static constexpr int kRows = 8 * NT, kSeqs = kPaMaxSeqs / kPdThreads;  // (sequences a thread counts)
    static constexpr bool kQShared = NT > 2;
    static constexpr int kE = NT <= 2 ? 2 : 1;

    static __device__ int item_steps(const PaParams &p, int b, PgSeq &seq, PaSpan<kPdStep> &span) {
        seq = pg_seq(p.b, p.c.page_size, b);
        if (seq.count * p.group > p.few_rows) seq.count = 0;  // the other kernel's
        span = pa_span<kPdStep>(max(seq.pos0, 0), seq.len - 1, p.window, p.sinks);
        return seq.count > 0 ? max(span.n, 1) + kPdItemCost : 0;  // rows that see nothing are written too
    }

    // Groups of kRows rows: items of their own, next to each other in the list (the second finds the codes
    // in L2).
    static __device__ __forceinline__ int groups(const PaParams &p, const PgSeq &seq) {
        return (seq.count * p.group + kRows - 1) / kRows;
    }

    // The piece that starts at unit u (< end, the CTA's end; `total` units in all).
    static __device__ void seek(const PaParams &p, const PdShared<NT> &sm, int u, int end, PdSeg &s) {
        int lo = 0, hi = p.b.num_seqs;  // the last sequence with prefix <= u
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (sm.prefix[mid] <= u) lo = mid;
            else hi = mid;
        }
        s.b = lo;
        const int units = item_steps(p, lo, s.seq, s.span), at = u - sm.prefix[lo];
        s.nb = units - kPdItemCost;
        const int item = at / units, of_head = groups(p, s.seq);
        s.h = item / of_head;
        s.row0 = (item - s.h * of_head) * kRows;
        s.first = sm.prefix[lo] + item * units + kPdItemCost;
        s.off = max(u - s.first, 0);
        s.n = min(s.nb, end - s.first) - s.off;  // not positive: only the item's cost lies before `end`
    }

    static __device__ void load_q(const PaParams &p, const PdSeg &s, int lane, int nt, uint32_t (&f)[16], float &factor) {
        const int r = s.row0 + nt * 8 + (lane >> 2), t = lane & 3;
        factor = 1.0f;
        if (r >= s.seq.count * p.group) {
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] = 0u;
            return;
        }
        const T *q = static_cast<const T *>(p.q) + (long)(s.seq.row0 + r / p.group) * p.q_stride +
                     (s.h * p.group + r % p.group) * kPgDim + 32 * t;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 v = reinterpret_cast<const uint4 *>(q)[i];
            f[4 * i] = v.x, f[4 * i + 1] = v.y, f[4 * i + 2] = v.z, f[4 * i + 3] = v.w;
        }
    }
    // bf16 queries become f16 with the row's largest value moved to [2^14, 2^15): exact down to 2^-31 of it
    // (f16's subnormals round eight bits from there on), 0 below 2^-39.  Returns what the products have to be
    // multiplied by.
    static __device__ float to_f16(uint32_t (&f)[16]) {
        if constexpr (sizeof(T) == 2 && !__is_same(T, __half)) {
            float amax = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(f[i] << 16)), fabsf(__uint_as_float(f[i] & 0xffff0000u))));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127 - 14, -120), 120);
            const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                f[i] = pg_pack2(__uint_as_float(f[i] << 16) * down, __uint_as_float(f[i] & 0xffff0000u) * down,
                                (const __half *)nullptr);
            return up;
        }
        return 1.0f;
    }

    static __device__ void write_row(const PaParams &p, const PdSeg &s, int r, int lane, float4 o, float m, float l) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        r += s.row0;
        const long at = (long)(s.seq.row0 + r / p.group) * p.query_heads + s.h * p.group + r % p.group;
        T *out = static_cast<T *>(p.out) + at * kPgDim;
        reinterpret_cast<uint2 *>(out)[lane] =
            make_uint2(pg_pack2(o.x * inv, o.y * inv, out), pg_pack2(o.z * inv, o.w * inv, out));
        if (p.lse && lane == 0) p.lse[at] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kPaLn2;
    }

    static __device__ void run(const PaParams &p, const CUtensorMap *kmap, const CUtensorMap *vmap, PdShared<NT> &sm) {
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
        launch_dependents();
        if (lane == 0) {
            for (int i = 0; i < kPdStages; ++i) mbar_init(&sm.full[warp][i], 1);
            fence_mbar_init();
        }
        grid_dependency_wait();
        const uint64_t deadline = globaltimer_ns() + kPaTimeoutNs;
        // prefix sums of the sequences' units: each thread takes four consecutive sequences
        int mine[kSeqs], sum = 0;
#pragma unroll
        for (int i = 0; i < kSeqs; ++i) {
            const int b = tid * (kSeqs) + i;
            PgSeq seq;
            PaSpan<kPdStep> span;
            mine[i] = b < p.b.num_seqs ? item_steps(p, b, seq, span) * p.c.kv_heads : 0;
            if (mine[i]) mine[i] *= groups(p, seq);
            sum += mine[i];
        }
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 31) sm.scan[warp] = incl;
        __syncthreads();
        int before = incl - sum, total = 0;
#pragma unroll
        for (int w = 0; w < kPdWarps; ++w) {
            if (w < warp) before += sm.scan[w];
            total += sm.scan[w];
        }
#pragma unroll
        for (int i = 0; i < kSeqs; ++i) {
            sm.prefix[tid * kSeqs + i] = before;
            before += mine[i];
        }
        __syncthreads();
        const int share = max((total + (int)gridDim.x - 1) / (int)gridDim.x, kPdWarps);
        const int u0 = min((long)share * blockIdx.x, (long)total), u1 = min(u0 + share, total);
        if (u0 >= u1) return;

        // ---- the copies: a cursor over this warp's steps, up to kPdStages ahead of the products
        PdSeg in;
        int in_u = u0, in_i = warp, in_base = 0, issued = 0;
        int row = -1;
        float ks = -1.0f, vs = 0.0f;
        bool in_open = false, in_done = false;
        auto issue = [&]() {
            while (!in_done) {
                if (!in_open) {
                    seek(p, sm, in_u, u1, in);
                    in_i = warp;
                    in_base = -1;
                    in_open = true;
                }
                if (in_i < in.n) break;
                in_u = in.first + in.nb;
                in_open = false;
                in_done = in_u >= u1;
            }
            if (in_done) return;
            const int at = in_i / kPdWarps;  // this warp's how-manieth step of the piece
            if (at >> 4 != in_base) {        // the pages and scales of its next 16 steps' groups, one a lane
                in_base = at >> 4;
                const int i = warp + kPdWarps * ((at & ~15) + (lane >> 1));
                row = -1;
                ks = -1.0f, vs = 0.0f;
                if (i < in.n) {
                    const int j = in.span.step(in.off + i) * kPdStep + 16 * (lane & 1);
                    int pid = -1;
                    // (a page that holds both groups counts for both, wherever the sequence ends in it)
                    if ((p.c.page_size == 16 ? j : j & ~31) < in.seq.len)
                        pid = p.b.page_table[(long)in.b * p.b.table_stride + j / p.c.page_size];
                    if (pid >= 0 && pid < p.c.num_pages) {
                        const int ph = pid * p.c.kv_heads + in.h;
                        row = ph * p.c.page_size + (j & (p.c.page_size - 1));
                        ks = p.c.k_scale[ph];
                        vs = p.c.v_scale[ph];
                    }
                }
            }
            const int st = issued % kPdStages;
            if ((lane >> 1) == (at & 15)) {  // the two lanes that know the step's groups
                const uint32_t pair = 3u << (lane & ~1);
                const int other = __shfl_xor_sync(pair, row, 1);
                uint64_t *bar = &sm.full[warp][st];
                if (!(lane & 1)) {
                    const int n = (row >= 0) + (other >= 0);
                    if (n) mbar_arrive_expect_tx(bar, n * kPdTile);
                    else mbar_arrive(bar);
                }
                __syncwarp(pair);
                // pages of 32 positions and more hold both groups: one copy each of keys and values
                if (row >= 0 && (p.c.page_size == 16 || !(lane & 1))) {
                    const int half = (lane & 1) * (kPdTile / 2);
                    pa_tma_2d(sm.ring[warp][st][0] + half, kmap, 0, row, bar);
                    pa_tma_2d(sm.ring[warp][st][1] + half, vmap, 0, row, bar);
                }
                // (the scales' reads may still be under way: the copies do not wait for them)
                reinterpret_cast<float2 *>(&sm.meta[warp][st])[lane & 1] = make_float2(ks, vs);
            }
            ++issued;
            in_i += kPdWarps;
        };
        for (int i = 0; i < kPdStages; ++i) issue();

        bool failed = false;
        int used = 0;
        for (int u = u0; u < u1;) {
            PdSeg s;
            seek(p, sm, u, u1, s);
            u = s.first + s.nb;
            if (s.n <= 0) continue;
            const int rows = min(s.seq.count * p.group - s.row0, kRows);
            uint32_t qf[kQShared ? 1 : NT][16];
            float qs[NT][2];  // the score's factor for this lane's two columns
            int pos[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float up = 1.0f;
                if (!kQShared || warp == nt) {
                    uint32_t f[16];
                    load_q(p, s, lane, nt, f, up);
                    up = to_f16(f) * fabsf(p.scale_log2);
                    if (p.scale_log2 < 0.0f) {  // the columns' factors stay >= 0
#pragma unroll
                        for (int i = 0; i < 16; ++i) f[i] ^= 0x80008000u;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if constexpr (kQShared) sm.q[i / 2][nt][lane][i & 1] = f[i];
                        else qf[nt][i] = f[i];
                    }
                    if constexpr (kQShared)
                        if (t == 0) sm.m[0][nt * 8 + g] = up;
                }
                if constexpr (!kQShared) {
                    qs[nt][0] = __shfl_sync(0xffffffffu, up, 8 * t);
                    qs[nt][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
                }
            }
            if constexpr (kQShared) {
                __syncthreads();
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) qs[nt][c] = sm.m[0][nt * 8 + 2 * t + c];
                __syncthreads();
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int r = nt * 8 + 2 * t + c;
                    pos[nt][c] = r < rows ? s.seq.pos0 + (s.row0 + r) / p.group : -1;
                }
            const int pos_lo = s.seq.pos0, pos_hi = s.seq.len - 1;
            float m[NT][2], l[NT][2], o[NT][8][4];  // per column; the maximum kPdNone before the first score
            float vref = 0.0f, vinv = 0.0f;  // the values' reference scale, 0 before the first
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int c = 0; c < 2; ++c) m[nt][c] = pos[nt][c] < 0 ? -kPdNone : kPdNone, l[nt][c] = 0.0f;  // (no row: P = 0)
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[nt][j][c] = 0.0f;
            }
            // The sums O to another reference.  Downwards they grow: by no more than takes the largest of them to
            // 2^100, for a page so far below it that f32 could not hold both.
            auto move = [&](float to) {
                float f = vref / to;
                if (f > 1.0f) {
                    float most = 0x1p-20f;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 8; ++j)
#pragma unroll
                            for (int c = 0; c < 4; ++c) most = fmaxf(most, fabsf(o[nt][j][c]));
                    most = fminf(warp_max_butterfly(most), 0x1p100f);  // (an infinity stays one)
                    f = fminf(f, 0x1p100f / __uint_as_float(__float_as_uint(most) & 0x7f800000u));
                    to = vref / f;
                }
                vref = to, vinv = 1.0f / to;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int c = 0; c < 4; ++c) o[nt][j][c] *= f;
            };
            for (int i = warp; i < s.n; i += kPdWarps, ++used) {
                const int st = used % kPdStages;
                if (!failed && !mbar_wait_bounded(&sm.full[warp][st], (used / kPdStages) & 1, deadline)) {
                    failed = true;
                    atomicExch(p.status, (uint32_t)MMRS_ERR_TIMEOUT);
                }
                __syncwarp();
                const float4 scales = sm.meta[warp][st];
                const float ksc[2] = {scales.x, scales.z}, vsc[2] = {scales.y, scales.w};
                const bool in0 = !(ksc[0] < 0.0f), in1 = !(ksc[1] < 0.0f);
                if (in0 || in1) {
                    const int j0 = s.span.step(s.off + i) * kPdStep;
                    const uint8_t *kt = sm.ring[warp][st][0], *vt = sm.ring[warp][st][1];
                    const bool whole = in0 && in1 && j0 + kPdStep - 1 <= pos_lo &&
                                       (p.window <= 0 || pos_hi - j0 < p.window || j0 + kPdStep <= p.sinks);
                    // kE groups at a time: both, where the registers allow it
#pragma unroll
                    for (int e0 = 0; e0 < 2; e0 += kE) {
                    float sc[kE][NT][4];
                    bool over = false;
                    // a column's factor: never 0, so that a masked score's -infinity stays one
                    auto factor = [&](int e, int nt, int c) { return fmaxf(qs[nt][c] * ksc[e0 + e], 1e-35f); };
                    auto largest = [&](int nt, int c) {
                        float mx = fmaxf(sc[0][nt][c], sc[0][nt][c + 2]) * factor(0, nt, c);
                        if constexpr (kE == 2)
                            mx = fmaxf(mx, fmaxf(sc[kE - 1][nt][c], sc[kE - 1][nt][c + 2]) * factor(kE - 1, nt, c));
                        return mx;
                    };
#pragma unroll
                    for (int e = 0; e < kE; ++e) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 4; ++c) sc[e][nt][c] = 0.0f;
                        uint32_t k0[8], k1[8];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const uint4 x = pd_lds(kt, 16 * (e0 + e) + g, 2 * t + c), y = pd_lds(kt, 16 * (e0 + e) + g + 8, 2 * t + c);
                            k0[4 * c] = x.x, k0[4 * c + 1] = x.y, k0[4 * c + 2] = x.z, k0[4 * c + 3] = x.w;
                            k1[4 * c] = y.x, k1[4 * c + 1] = y.y, k1[4 * c + 2] = y.z, k1[4 * c + 3] = y.w;
                        }
#pragma unroll
                        for (int ks8 = 0; ks8 < 8; ++ks8) {
                            uint32_t a0, a1, a2, a3;
                            pg_e4m3x4_to_half2(k0[ks8], a0, a2);
                            pg_e4m3x4_to_half2(k1[ks8], a1, a3);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                if constexpr (kQShared) {
                                    const uint2 b = *reinterpret_cast<const uint2 *>(sm.q[ks8][nt][lane]);
                                    pd_mma(sc[e][nt], a0, a1, a2, a3, b.x, b.y);
                                } else {
                                    pd_mma(sc[e][nt], a0, a1, a2, a3, qf[nt][2 * ks8], qf[nt][2 * ks8 + 1]);
                                }
                            }
                        }
                    }
                    if (!whole) {
#pragma unroll
                        for (int e = 0; e < kE; ++e)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int c = 0; c < 4; ++c)
                                    if (!(e0 + e ? in1 : in0) ||
                                        !pa_sees(j0 + 16 * (e0 + e) + g + (c >> 1) * 8, pos[nt][c & 1], p.window, p.sinks))
                                        sc[e][nt][c] = -INFINITY;
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c)
                            over = over || largest(nt, c) > m[nt][c] + kPdLazy;
                    if (__any_sync(0xffffffffu, over)) {
                        if (vref == 0.0f) {  // the first page's scale, here (O is zero) rather than by a branch of its own
                            vref = kE == 2 ? fmaxf(vsc[0], vsc[1]) : vsc[e0];
                            vinv = vref > 0.0f ? 1.0f / vref : 0.0f;
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                float mx = largest(nt, c);
                                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                                mx = fmaxf(mx, m[nt][c]);
                                const float fac = pa_exp2(m[nt][c] - mx);
                                m[nt][c] = mx;
                                l[nt][c] *= fac;
#pragma unroll
                                for (int j = 0; j < 8; ++j) o[nt][j][c] *= fac, o[nt][j][c + 2] *= fac;
                            }
                    }
                    uint32_t pb[kE][NT][2];
#pragma unroll
                    for (int e = 0; e < kE; ++e) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            float p4[4];
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const float f = factor(e, nt, c);
                                p4[c] = pa_exp2(fmaf(sc[e][nt][c], f, -m[nt][c]));
                                p4[c + 2] = pa_exp2(fmaf(sc[e][nt][c + 2], f, -m[nt][c]));
                                l[nt][c] += p4[c] + p4[c + 2];
                            }
                            pb[e][nt][0] = pd_transpose(pg_pack2(p4[0], p4[1], (const __half *)nullptr));
                            pb[e][nt][1] = pd_transpose(pg_pack2(p4[2], p4[3], (const __half *)nullptr));
                        }
                    }
#pragma unroll
                    for (int e = 0; e < kE; ++e) {
                        // The values' scale enters P relative to the warp's reference, which follows the pages up, and
                        // down where one lies far below it (P times the ratio keeps f16's eleven bits down to 2^-8); a
                        // page without any weight, or whose values are all zero, does not move it.
                        float ratio = vsc[e0 + e] * vinv;
                        if (__float_as_uint(ratio) - __float_as_uint(kPdUnder) >= __float_as_uint(2.0f) - __float_as_uint(kPdUnder)) {
                            uint32_t some = 0;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) some |= pb[e][nt][0] | pb[e][nt][1];
                            ratio = 0.0f;
                            if (vsc[e0 + e] > 0.0f && __any_sync(0xffffffffu, some != 0)) {
                                move(vsc[e0 + e]);
                                ratio = vsc[e0 + e] * vinv;
                            }
                        }
                        // (a product of halves: exact for scales that are powers of two)
                        const __half2 vr = __float2half2_rn(ratio);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const __half2 z = __hmul2(*reinterpret_cast<const __half2 *>(&pb[e][nt][c]), vr);
                                pb[e][nt][c] = *reinterpret_cast<const uint32_t *>(&z);
                            }
                        uint4 v4[4];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int r = 2 * t + (c & 1) + (c >> 1) * 8;
                            v4[c] = pd_lds(vt, 16 * (e0 + e) + r, g);
                            // slots past the sequence's end may hold anything
                            if (!whole && (!(e0 + e ? in1 : in0) || j0 + 16 * (e0 + e) + r >= s.seq.len)) v4[c] = make_uint4(0u, 0u, 0u, 0u);
                        }
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const uint32_t x[4] = {reinterpret_cast<const uint32_t *>(&v4[0])[w],
                                                   reinterpret_cast<const uint32_t *>(&v4[1])[w],
                                                   reinterpret_cast<const uint32_t *>(&v4[2])[w],
                                                   reinterpret_cast<const uint32_t *>(&v4[3])[w]};
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                const uint32_t sel = half ? 0x7362u : 0x5140u;
                                uint32_t a0, a1, a2, a3;
                                pg_e4m3x4_to_half2(__byte_perm(x[0], x[1], sel), a0, a1);
                                pg_e4m3x4_to_half2(__byte_perm(x[2], x[3], sel), a2, a3);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
                                    pd_mma(o[nt][2 * w + half], a0, a1, a2, a3, pb[e][nt][0], pb[e][nt][1]);
                            }
                        }
                    }
                    }
                }
                __syncwarp();
                issue();
            }
            // ---- the warps' results of this piece
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], x);
                    if (g == 0) sm.m[warp][nt * 8 + 2 * t + c] = m[nt][c], sm.l[warp][nt * 8 + 2 * t + c] = l[nt][c];
                }
            const int c0 = s.first / share, c1 = (s.first + s.nb - 1) / share;  // the parts that hold steps of it
            float *slot = p.partials + ((size_t)blockIdx.x * 2 + ((int)blockIdx.x == c0 ? 1 : 0)) * (32 * (kPgDim + 2));
            __syncthreads();
            // every warp's sums to the common maximum; the upper half of the warps' into the lower's
            auto sums = [&](int nt, int c, int j) {
                return reinterpret_cast<float4 *>(&sm.o[warp % (kPdWarps / 2)][nt * 8 + 2 * t + c][16 * g + 2 * j]);
            };
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int r = nt * 8 + 2 * t + c;
                    float top = kPdNone;
#pragma unroll
                    for (int w = 0; w < kPdWarps; ++w) top = fmaxf(top, sm.m[w][r]);
                    const float f = pa_exp2(m[nt][c] - top) * vref;
#pragma unroll
                    for (int j = 0; j < 8; ++j) o[nt][j][c] *= f, o[nt][j][c + 2] *= f;
                    if (warp >= kPdWarps / 2) {
#pragma unroll
                        for (int j = 0; j < 8; j += 2)
                            *sums(nt, c, j) = make_float4(o[nt][j][c], o[nt][j][c + 2], o[nt][j + 1][c], o[nt][j + 1][c + 2]);
                    }
                }
            __syncthreads();
            if (warp < kPdWarps / 2) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int j = 0; j < 8; j += 2) {
                            const float4 x = *sums(nt, c, j);
                            *sums(nt, c, j) = make_float4(o[nt][j][c] + x.x, o[nt][j][c + 2] + x.y, o[nt][j + 1][c] + x.z,
                                                          o[nt][j + 1][c + 2] + x.w);
                        }
            }
            __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int r = nt * 8 + warp;  // eight warps, eight rows of each group
                float top = kPdNone, sum_l = 0.0f;
#pragma unroll
                for (int w = 0; w < kPdWarps; ++w) top = fmaxf(top, sm.m[w][r]);
                float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kPdWarps; ++w) sum_l += sm.l[w][r] * pa_exp2(sm.m[w][r] - top);
#pragma unroll
                for (int w = 0; w < kPdWarps / 2; ++w) {
                    const float4 x = *reinterpret_cast<const float4 *>(&sm.o[w][r][4 * lane]);
                    acc.x += x.x, acc.y += x.y, acc.z += x.z, acc.w += x.w;
                }
                if (r < rows) {
                    if (c0 == c1) {
                        write_row(p, s, r, lane, acc, top, sum_l);
                    } else {
                        reinterpret_cast<float4 *>(slot + r * kPgDim)[lane] = acc;
                        if (lane == 0) slot[32 * kPgDim + r] = top, slot[32 * kPgDim + 32 + r] = sum_l;
                    }
                }
            }
            __syncthreads();
            if (c0 != c1) {
                uint32_t *counter = p.counters + c0;
                if (tid == 0) {
                    __threadfence();
                    sm.last = atomicAdd(counter, 1u) == (uint32_t)(c1 - c0);
                    __threadfence();
                }
                __syncthreads();
                if (sm.last) {
                    // this warp's rows together, so that their reads of L2 overlap
                    constexpr int kMine = (kRows + kPdWarps - 1) / kPdWarps;
                    auto at = [&](int c) {
                        return p.partials + ((size_t)c * 2 + (c == c0 ? 1 : 0)) * (32 * (kPgDim + 2));
                    };
                    float top[kMine], sum_l[kMine];
                    float4 acc[kMine];
#pragma unroll
                    for (int i = 0; i < kMine; ++i) {
                        top[i] = kPdNone, sum_l[i] = 0.0f;
                        acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    }
                    for (int cb = c0; cb <= c1; cb += 32) {  // 32 parts' factors, one a lane; then their rows
                        float f[kMine], lc[kMine];
#pragma unroll
                        for (int i = 0; i < kMine; ++i) {
                            f[i] = kPdNone, lc[i] = 0.0f;
                            if (cb + lane <= c1 && warp + i * kPdWarps < rows) {
                                const float *a = at(cb + lane) + 32 * kPgDim + warp + i * kPdWarps;
                                f[i] = __ldcg(a);
                                lc[i] = __ldcg(a + 32);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < kMine; ++i) {
                            const float now = fmaxf(top[i], warp_max_butterfly(f[i])), less = pa_exp2(top[i] - now);
                            top[i] = now;
                            f[i] = pa_exp2(f[i] - now);
                            lc[i] *= f[i];
                            sum_l[i] *= less;
                            acc[i].x *= less, acc[i].y *= less, acc[i].z *= less, acc[i].w *= less;
                        }
                        const int n = min(32, c1 - cb + 1);
#pragma unroll kMine == 1 ? 8 : 4
                        for (int c = 0; c < n; ++c) {
#pragma unroll
                            for (int i = 0; i < kMine; ++i) {
                                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                                if (warp + i * kPdWarps < rows)
                                    x = __ldcg(reinterpret_cast<const float4 *>(at(cb + c) + (warp + i * kPdWarps) * kPgDim) + lane);
                                const float fc = __shfl_sync(0xffffffffu, f[i], c);
                                sum_l[i] += __shfl_sync(0xffffffffu, lc[i], c);
                                acc[i].x += fc * x.x, acc[i].y += fc * x.y, acc[i].z += fc * x.z, acc[i].w += fc * x.w;
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kMine; ++i)
                        if (warp + i * kPdWarps < rows) write_row(p, s, warp + i * kPdWarps, lane, acc[i], top[i], sum_l[i]);
                    if (tid == 0) *counter = 0u;
                }
            }
        }
        if (failed)  // copies that came late must not land in another block's memory
            for (int i = used < kPdStages ? 0 : used - kPdStages; i < issued; ++i)
                mbar_wait_bounded(&sm.full[warp][i % kPdStages], (i / kPdStages) & 1, deadline + kPaTimeoutNs);
    }
};

template <int NT, typename T>
__global__ void __launch_bounds__(kPdThreads, 1)
    paged_attend_decode_kernel(const __grid_constant__ PaParams p, const __grid_constant__ CUtensorMap kmap,
                               const __grid_constant__ CUtensorMap vmap) {
    extern __shared__ uint8_t raw[];
    PdShared<NT> &sm = *reinterpret_cast<PdShared<NT> *>(raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u));
    PdKernel<NT, T>::run(p, &kmap, &vmap, sm);
}

template <int NT, typename T>
int pd_launch(const PaParams &p, const CUtensorMap &k, const CUtensorMap &v, cudaStream_t s) {
    constexpr size_t kPdSmem = sizeof(PdShared<NT>) + 1024;
    static_assert(kPdSmem <= 227 * 1024, "shared memory");
    static std::once_flag once[64];
    static cudaError_t set_rc[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return MMRS_ERR_LAUNCH;
    std::call_once(once[dev], [dev] {
        set_rc[dev] = cudaFuncSetAttribute(paged_attend_decode_kernel<NT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)kPdSmem);
    });
    if (set_rc[dev] != cudaSuccess) return MMRS_ERR_LAUNCH;
    return pg_launch(paged_attend_decode_kernel<NT, T>, (unsigned)pa_sm_count(), kPdThreads, kPdSmem, s, p, k, v);
}

template <typename T>
int pd_launch_rows(const PaParams &p, const CUtensorMap &k, const CUtensorMap &v, cudaStream_t s) {
    // the fewest items a sequence, of equal size; next to prompts in one call, where single tokens or drafts
    // may be there, 16 rows
    const int most = p.b.max_q * p.group, items = (most + kPaDecodeRows - 1) / kPaDecodeRows;
    const int rows = p.mixed ? 16 : (most + items - 1) / items;
    if (rows <= 8) return pd_launch<1, T>(p, k, v, s);
    if (rows <= 16) return pd_launch<2, T>(p, k, v, s);
    if (rows <= 24) return pd_launch<3, T>(p, k, v, s);
    return pd_launch<4, T>(p, k, v, s);
}

}  // namespace

int pa_launch_decode(const PaParams &p, const CUtensorMap &k, const CUtensorMap &v, int type, cudaStream_t s) {
    return type == MMRS_TYPE_F16 ? pd_launch_rows<__half>(p, k, v, s) : pd_launch_rows<__nv_bfloat16>(p, k, v, s);
}

}  // namespace mmrs
