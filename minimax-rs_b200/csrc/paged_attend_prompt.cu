// Paged attention of many rows: prompt chunks, and drafts of more than kPaFewRows rows a KV head.
//
// Here every code is used by hundreds of rows, so the kernel is bound by arithmetic: 4 * 128 flops
// a (row, position) on the tensor cores and one exponential, and the two weigh about the same on
// an SM (a 128x128 tile takes 1024 cycles of either).  The rows of a KV head (new tokens x query
// heads of its group) are packed 256 to an item, two M = 128 tiles whose softmax and products
// alternate, so that one tile's exponentials run under the other's products:
//   warps 0-3, 4-7   softmax of tile 0, 1, one thread a row: S from tensor memory, running maximum
//                    and sum, P (f16) back into S's columns, and the epilogue
//   warps 8-11       K and V codes from global memory through registers (one tile ahead), e4m3 to
//                    f16 (exact), into the operand layouts
//   warps 12, 13     issue S = Q K^T (both operands in shared memory) and O += P V (P in tensor
//                    memory), kind::f16, for tile 0, 1
// A tile's scores go through in halves of 64 positions, each with its own barriers: while one half's
// exponentials run, the other half's product does (1783 -> 1605 us at the prompt below).
// Operand tiles are without swizzle: 16-byte pieces (8 columns of one row) with the eight rows of a
// core matrix next to each other; the same form serves K (K-major) and V (its columns are the
// product's N, so the tile is read MN-major).
//
// Scales: a page's key scale multiplies its columns' scores in the exponent's FMA.  Its value scale,
// relative to a reference, multiplies the values on their way to f16 (exact for the powers of two that the
// append writes, one rounding otherwise).  Neither costs the softmax anything an element.  The reference is the
// piece's, from its largest scale; where scales lie more than 2^22 apart, it is each tile's, and O is rescaled
// with it as with the maximum.  (One reference for the piece and nothing else took 1430 us instead of 1447 at the
// prompt below, and lost the values of pages 2^26 below the largest.)  The running maximum moves only when it
// grows by more than 2^8 (P stays below f16's range), which leaves O alone on almost every tile.
//
// Masks: a half that all of a warp's rows see whole costs one vote; one that none sees is left out; else
// 64 visibility bits a row choose between scores in registers (a pass through tensor memory of their
// own, with the queries read a row a lane: 228 us instead of 176 for the windowed prompts below).
//
// Work: the (item, 128-position tile) pairs of all sequences form one list, of which each CTA (one
// per SM) takes an equal contiguous part; an item cut by that gets its pieces joined through the
// workspace by the CTA that finishes last, in order.
//
// Measured: 4096 tokens behind 12288 others, 48 + 8 heads, f16: 1447 us from a cold start (997 TFLOP/s,
// 0.61 of what the library's largest product reaches), some 1690 us under the power limit.  The tensor
// cores are busy 40 % of the time and the exponential units 45 %: what is left is the chain of one
// half, scores -> maximum -> exponentials -> P -> product, some 2500 cycles with two tiles to fill it
// (half of the scores, three quarters of P V or all exponentials left out: 2 % less).  Five
// ragged prompts of 1 to 2049 tokens with a window of 511, 32 + 4 heads: 160 us, of which 80 us are
// full tiles' and most of the rest items' beginnings, ends and masked halves.
#include "paged_attend.cuh"
#include "umma.cuh"

#include <mutex>

namespace mmrs {
namespace {

constexpr int kPpThreads = 16 * 32;  // four warpgroups; the last has two working warps
constexpr int kPpKeys = 128;                 // positions of a tile
constexpr int kPpRows = 256;                 // rows of an item
constexpr int kPpTile = 128 * kPgDim * 2;    // bytes of an operand tile
constexpr int kPpSlice = 128 * 16;           // bytes between 8-column slices of a tile
constexpr int kPpStages = 2;
constexpr int kPpScales = 4;                 // tiles whose scales are kept
constexpr float kPpLazy = 8.0f;              // log2 of how far P may exceed 1
// The largest value scale in units of the reference: codes (up to 448) times it stay in f16's range.  A code times
// the least scale that kPpExact allows for keeps its bits (e4m3's subnormals end at 2^-9, f16's at 2^-24).
constexpr float kPpAbove = 128.0f;
constexpr float kPpExact = 0x1p-22f;  // least over largest
constexpr float kPpDown = 0x1p-60f;   // how far below the largest one met the reference follows (O stays below 2^104)
constexpr int kPpConvWarp0 = 8, kPpMmaWarp = 12;

struct alignas(16) PpScale {  // of the eight 16-position groups of a tile
    float k[8];  // key scale; < 0: the group's page holds nothing
    float vref;  // what the tile's values are relative to
};
struct PpShared {
    uint8_t q[2][kPpTile], k[kPpStages][kPpTile], v[kPpStages][kPpTile];
    float row_top[kPpRows], row_inv[kPpRows];  // of an item's rows while its pieces are joined
    PpScale sc[kPpScales];
    float2 vrange[4];  // largest and least value scale of a converter warp's groups
    float high[4], unit[4];  // a converter warp's reference, and pp_follow's largest scale (negative: one reference a piece)
    int prefix[kPaMaxSeqs + 1];
    uint64_t q_full[2], s_full[2][2], p_full[2][2], o_done[2][2];  // [row tile][half]
    uint64_t k_full[kPpStages], k_empty[kPpStages], v_full[kPpStages], v_empty[kPpStages], sc_full[kPpScales];
    uint64_t mdone[2];
    uint32_t tmem;
    int abort, last;
};
constexpr size_t kPpSmem = sizeof(PpShared) + 128;
static_assert(kPpSmem <= 227 * 1024, "shared memory");

constexpr uint32_t kPpIdesc = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);  // f16 x f16 -> f32, 128 x 128
constexpr uint32_t kPpIdescV = kPpIdesc | (1u << 16);  // B read MN-major
constexpr uint32_t kPpIdescS = (1u << 4) | ((64u >> 3) << 17) | ((128u >> 4) << 24);  // 128 x 64
constexpr uint32_t kColS = 0, kColO = 256;

// Descriptors as their 32-bit halves (umma_smem_desc): only the low one moves with the address.
__device__ __forceinline__ uint32_t pp_desc_lo(uint32_t saddr, uint32_t lbo) {
    return (saddr >> 4) | (lbo >> 4) << 16;
}
constexpr uint32_t pp_desc_hi(uint32_t sbo) { return (sbo >> 4) | 1u << 14; }
__device__ __forceinline__ void pp_mma_ss(uint32_t d, uint32_t alo, uint32_t ahi, uint32_t blo, uint32_t bhi,
                                          uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
        "setp.ne.b32 p, %6, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t}" ::"r"(d),
        "r"(alo), "r"(ahi), "r"(blo), "r"(bhi), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void pp_mma_ts(uint32_t d, uint32_t a, uint32_t blo, uint32_t bhi, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(blo), "r"(bhi), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void pp_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t *u = reinterpret_cast<uint32_t *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
        "%30,%31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
          "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
          "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
          "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
        : "r"(taddr));
}
__device__ __forceinline__ void pp_st16(uint32_t taddr, const uint32_t (&u)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(
            u[0]),
        "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]),
        "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(taddr)
        : "memory");
}
// Waits for the loads; `v` passes through so that no use of it moves before the wait.
__device__ __forceinline__ void pp_hold32(float *v) {
    asm volatile(""
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                   "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]));
    asm volatile(""
                 : "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]),
                   "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31]));
}
__device__ __forceinline__ void pp_wait_ld(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    pp_hold32(v);
}
// Two f32 in one register pair: one instruction for both.
__device__ __forceinline__ uint64_t pp_pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void pp_split(uint64_t r, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t pp_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t pp_add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// 2^x of both halves on the FMA units: x = n + f, |f| <= 1/2, 2^f by a degree-4 polynomial (relative
// error below 2.7e-6 in f32, the least-maximum fit of 2^f; P keeps 2^-11), times 2^n made from n's
// bits.  The special-function units give a warp four results a cycle; one pair in four this way takes
// 20 % off a tile's exponentials (1474 -> 1108 cycles for one warp of a scheduler, 2380 -> 1908 for
// two), and three in eight no more.  x below -126 counts as -126, NaN stays NaN.
__device__ __forceinline__ uint64_t pp_exp2_fma(uint64_t x) {
    float a, b;
    pp_split(x, a, b);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-126.0f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-126.0f));
    x = pp_pair(a, b);
    const uint64_t r = pp_add2(x, pp_pair(12582912.0f, 12582912.0f));  // 1.5 * 2^23: rounds to whole numbers
    const uint64_t f = pp_fma2(pp_add2(r, pp_pair(-12582912.0f, -12582912.0f)), pp_pair(-1.0f, -1.0f), x);
    uint64_t y = pp_fma2(f, pp_pair(0.009570102f, 0.009570102f), pp_pair(0.05591786f, 0.05591786f));
    y = pp_fma2(y, f, pp_pair(0.24024744f, 0.24024744f));
    y = pp_fma2(y, f, pp_pair(0.6931218f, 0.6931218f));
    y = pp_fma2(y, f, pp_pair(0.9999993f, 0.9999993f));
    pp_split(r, a, b);
    a = __int_as_float((__float_as_int(a) << 23) + 0x3f800000), b = __int_as_float((__float_as_int(b) << 23) + 0x3f800000);
    uint64_t z;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(z) : "l"(y), "l"(pp_pair(a, b)));
    return z;
}
__device__ __forceinline__ void pp_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The columns of a 64-column half that a row sees, as bits: x <= at, with a window (x > at - window or
// x < first), and the groups of 16 whose page holds something.
__device__ __forceinline__ uint64_t pp_upto(int n) { return n < 0 ? 0ull : n >= 63 ? ~0ull : (2ull << n) - 1; }
__device__ __forceinline__ uint64_t pp_sees(int at, int window, int first, const float4 &ks) {
    uint64_t see = pp_upto(at);
    if (window > 0) see &= ~pp_upto(at - window) | pp_upto(first - 1);
    if (ks.x < 0.0f) see &= ~0xffffull;
    if (ks.y < 0.0f) see &= ~(0xffffull << 16);
    if (ks.z < 0.0f) see &= ~(0xffffull << 32);
    if (ks.w < 0.0f) see &= ~(0xffffull << 48);
    return see;
}

// A row of O times f.
__device__ __forceinline__ void pp_scale_o(uint32_t to, float f) {
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        float v[32];
        pp_ld32(to + 32 * c, v);
        pp_wait_ld(v);
        uint32_t w[2][16];
#pragma unroll
        for (int x = 0; x < 32; ++x) w[x >> 4][x & 15] = __float_as_uint(v[x] * f);
        pp_st16(to + 32 * c, w[0]);
        pp_st16(to + 32 * c + 16, w[1]);
    }
    pp_wait_st();
}

// Bounded wait of one role: false when about two seconds have passed (2^20 sleeps of at most 2 us) or
// another role has given up.  The warp sleeps in hardware until the phase ends: a spinning one takes
// the path that the exponentials and shared memory need.
__device__ __forceinline__ bool pp_wait(uint64_t *bar, uint32_t parity, PpShared &sm, const PaParams &p) {
    if (mbar_test_wait(bar, parity)) return true;
#pragma unroll 1
    for (int n = 0; n < (1 << 20); ++n) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(2000u)
            : "memory");
        if (ok) return true;
        if (*reinterpret_cast<volatile int *>(&sm.abort)) return false;
    }
    *reinterpret_cast<volatile int *>(&sm.abort) = 1;
    atomicExch(p.status, (uint32_t)MMRS_ERR_TIMEOUT);
    return false;
}

// The same for a whole warp, with one answer.
__device__ __forceinline__ bool pp_wait_warp(uint64_t *bar, uint32_t parity, PpShared &sm, const PaParams &p) {
    return __all_sync(0xffffffffu, pp_wait(bar, parity, sm, p)) != 0;
}

// An item's piece: sequence b, KV head h, rows [row0, row0 + rows) of the sequence's packed rows,
// tiles [off, off + n) of the item's nb.
struct PpSeg {
    int b, h, row0, rows, off, n, nb;
    PgSeq seq;
    PaSpan<kPpKeys> span;
};

__device__ __forceinline__ int pp_tiles(const PaParams &p, const PgSeq &seq, int rt, PaSpan<kPpKeys> &span) {
    const int total = seq.count * p.group, last = min((rt + 1) * kPpRows, total) - 1;
    const int lo = max(seq.pos0 + rt * kPpRows / p.group, 0), hi = seq.pos0 + last / p.group;
    span = pa_span<kPpKeys>(lo, max(hi, -1), p.window, p.sinks);
    return max(span.n, 1);  // rows that see nothing are written too
}
// Units of one KV head of a sequence (whole warp); none of one that is the decode kernel's.
__device__ int pp_seq_units(const PaParams &p, const PgSeq &seq, int lane) {
    const int tiles = seq.count * p.group <= p.few_rows ? 0 : (seq.count * p.group + kPpRows - 1) / kPpRows;
    int sum = 0;
    PaSpan<kPpKeys> span;
#pragma unroll 1
    for (int rt = lane; rt < tiles; rt += 32) sum += pp_tiles(p, seq, rt, span);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}
// The piece that starts at unit u (whole warp).
__device__ void pp_seek(const PaParams &p, const PpShared &sm, int u, int end, int lane, PpSeg &s) {
    int lo = 0, hi = p.b.num_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (sm.prefix[mid] <= u) lo = mid;
        else hi = mid;
    }
    s.b = lo;
    s.seq = pg_seq(p.b, p.c.page_size, lo);
    const int per_head = (sm.prefix[lo + 1] - sm.prefix[lo]) / p.c.kv_heads;
    int at = u - sm.prefix[lo];
    s.h = at / per_head;
    at -= s.h * per_head;
    const int tiles = (s.seq.count * p.group + kPpRows - 1) / kPpRows;
    int rt = 0, before = 0;
#pragma unroll 1
    for (int r0 = 0; r0 < tiles; r0 += 32) {
        PaSpan<kPpKeys> span;
        const int n = r0 + lane < tiles ? pp_tiles(p, s.seq, r0 + lane, span) : 0;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, before + incl > at);
        if (past) {
            const int l = __ffs(past) - 1;
            rt = r0 + l;
            s.off = at - before - __shfl_sync(0xffffffffu, incl - n, l);
            break;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    s.nb = pp_tiles(p, s.seq, rt, s.span);
    s.n = min(s.nb - s.off, end - u);
    s.row0 = rt * kPpRows;
    s.rows = min(kPpRows, s.seq.count * p.group - s.row0);
}
// The piece after s, which ends an item at unit u (whole warp): the lookup of pp_seek, some 2500 cycles,
// only where a new sequence begins.
__device__ void pp_next(const PaParams &p, const PpShared &sm, int u, int end, int lane, PpSeg &s) {
    int rt = s.row0 / kPpRows + 1, h = s.h;
    if (rt * kPpRows >= s.seq.count * p.group) rt = 0, ++h;
    if (h >= p.c.kv_heads) {
        pp_seek(p, sm, u, end, lane, s);
        return;
    }
    s.h = h, s.off = 0;
    s.nb = pp_tiles(p, s.seq, rt, s.span);
    s.n = min(s.nb, end - u);
    s.row0 = rt * kPpRows;
    s.rows = min(kPpRows, s.seq.count * p.group - s.row0);
}

// A read that leaves the L1 alone.
__device__ __forceinline__ uint4 pp_ldg(const uint8_t *at) {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(at));
    return r;
}

// ---- warps 8-11: codes to f16 operand tiles ------------------------------------------------------
// Thread: key (lane & 7) of each of its warp's four 8-key groups, 16-code chunks (lane >> 3) and + 4.
template <bool kScaled>
__device__ __forceinline__ void pp_store_tile(uint8_t *tile, const uint4 (&raw)[8], int w, int lane, const __half2 *rel) {
#pragma unroll
    for (int it = 0; it < 8; ++it) {
        const int group = w * 4 + (it >> 1), chunk = (it & 1) * 4 + (lane >> 3);
        uint8_t *at = tile + 2 * chunk * kPpSlice + group * 128 + (lane & 7) * 16;
        const uint4 r = raw[it];
        uint4 a, b;
        pg_e4m3x4_to_half2(r.x, a.x, a.y), pg_e4m3x4_to_half2(r.y, a.z, a.w);
        pg_e4m3x4_to_half2(r.z, b.x, b.y), pg_e4m3x4_to_half2(r.w, b.z, b.w);
        if constexpr (kScaled) {
            const __half2 f = rel[it >> 2];
            auto times = [&](uint32_t &x) {
                const __half2 y = __hmul2(*reinterpret_cast<const __half2 *>(&x), f);
                x = *reinterpret_cast<const uint32_t *>(&y);
            };
            times(a.x), times(a.y), times(a.z), times(a.w), times(b.x), times(b.y), times(b.z), times(b.w);
        }
        *reinterpret_cast<uint4 *>(at) = a;
        *reinterpret_cast<uint4 *>(at + kPpSlice) = b;
    }
}

// The reference for a largest scale (never 0).
__device__ __forceinline__ float pp_unit(float scale) { return fmaxf(scale / kPpAbove, 0x1p-126f); }

// A tile of a piece whose value scales lie far apart, at position `at` (whole warp): its reference goes to *unit, which
// has the last one's, and the ratios of the converter warp's two groups are returned.  high: the largest scale of
// the tiles so far, 0 before the first.
__device__ __noinline__ float2 pp_follow(const PaParams &p, int b, int head, int at, int len, float *unit, float *high) {
    const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) - kPpConvWarp0, j = at + lane * 16;
    float x = 0.0f;
    if (lane < 8 && j < len) {
        const int page = p.b.page_table[(long)b * p.b.table_stride + j / p.c.page_size];
        if (page >= 0 && page < p.c.num_pages) x = p.c.v_scale[(long)page * p.c.kv_heads + head];
    }
    const float most = warp_max_butterfly(x), least = -warp_max_butterfly(x > 0.0f ? -x : -INFINITY), was = *high;
    float vref = *unit;
    if (most > 0.0f && (was == 0.0f || most > vref * kPpAbove || least < vref * (kPpAbove * kPpExact))) {
        vref = pp_unit(fmaxf(most, was * kPpDown));
        __syncwarp();
        if (lane == 0) *unit = vref, *high = fmaxf(was, most);
    }
    __syncwarp();
    x /= vref;
    return make_float2(__shfl_sync(0xffffffffu, x, 2 * w), __shfl_sync(0xffffffffu, x, 2 * w + 1));
}

__device__ void pp_convert(const PaParams &p, PpShared &sm, int u0, int u1) {
    const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) - kPpConvWarp0;
    int tile = 0;
    bool ok = true;  // after a failed wait only the barriers among these warps go on
    PpSeg s;
#pragma unroll 1
    for (int u = u0; u < u1;) {
        if (u == u0) pp_seek(p, sm, u, u1, lane, s);
        else pp_next(p, sm, u, u1, lane, s);
        const int ps = p.c.page_size;
        // the pages and scales of this warp's two 16-position groups in 16 tiles, one a lane
        int pid = -1;
        float ks = 0.0f, vs = 0.0f;
        auto fetch = [&](int base) {
            const int i = base + (lane >> 1);
            pid = -1, ks = -1.0f, vs = 0.0f;
            if (i < s.n) {
                const int j = s.span.step(s.off + i) * kPpKeys + w * 32 + (lane & 1) * 16;
                if (j < s.seq.len) pid = p.b.page_table[(long)s.b * p.b.table_stride + j / ps];
                if (pid >= p.c.num_pages) pid = -1;
                if (pid >= 0) {
                    ks = p.c.k_scale[(long)pid * p.c.kv_heads + s.h];
                    vs = p.c.v_scale[(long)pid * p.c.kv_heads + s.h];
                }
            }
        };
        float high = 0.0f, least = INFINITY;  // of the piece's value scales, zeros aside
        auto range = [&](float x) { high = fmaxf(high, x), least = fminf(least, x > 0.0f ? x : INFINITY); };
#pragma unroll 1
        for (int base = (s.n - 1) & ~15; base >= 0; base -= 16) {  // the first sixteen last: they come next
            fetch(base);
            range(vs);
        }
        high = warp_max_butterfly(high), least = -warp_max_butterfly(-least);
        named_sync(2, 128);
        if (lane == 0) sm.vrange[w] = make_float2(high, least);
        named_sync(2, 128);
#pragma unroll
        for (int x = 0; x < 4; ++x) high = fmaxf(high, sm.vrange[x].x), least = fminf(least, sm.vrange[x].y);
        // one reference for the piece, or, where that would cost values, the tiles' own
        high = high > 0.0f ? high : kPpAbove;
        __syncwarp();
        if (lane == 0) sm.high[w] = least < high * kPpExact ? 0.0f : -1.0f, sm.unit[w] = pp_unit(high);
        __syncwarp();
        vs /= sm.unit[w];  // from here on the ratio
        uint4 kr[8], vr[8];
        // this thread's rows and columns in its two 16-position groups of tile i
        long at[2];
        int left[2];
        auto place = [&](int i) {
            const int j = s.span.step(s.off + i) * kPpKeys + w * 32;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int page = __shfl_sync(0xffffffffu, pid, (i & 15) * 2 + g);
                at[g] = (((long)page * p.c.kv_heads + s.h) * ps + ((j + 16 * g) & (ps - 1)) + (lane & 7)) * kPgDim +
                        16 * (lane >> 3);
                left[g] = page < 0 ? 0 : s.seq.len - (j + 16 * g + (lane & 7));  // > 8 u: row u of it is in the sequence
            }
        };
        auto load = [&](const void *codes, uint4 (&r)[8]) {
            const uint8_t *base = static_cast<const uint8_t *>(codes);
#pragma unroll
            for (int it = 0; it < 8; ++it) {
                const int g = it >> 2, u = (it >> 1) & 1;
                r[it] = make_uint4(0u, 0u, 0u, 0u);  // slots past the sequence's end may hold anything
                if (left[g] > 8 * u) r[it] = pp_ldg(base + at[g] + u * 8 * kPgDim + (it & 1) * 64);
            }
        };
        place(0);
        load(p.c.k, kr);
        load(p.c.v, vr);
#pragma unroll 1
        for (int i = 0; ok && i < s.n; ++i, ++tile) {
            const int st = tile % kPpStages, use = tile / kPpStages;
            PpScale &sc = sm.sc[tile % kPpScales];
            if ((lane >> 1) == (i & 15)) sc.k[2 * w + (lane & 1)] = ks;
            float2 r = make_float2(__shfl_sync(0xffffffffu, vs, (i & 15) * 2), __shfl_sync(0xffffffffu, vs, (i & 15) * 2 + 1));
            if (sm.high[w] >= 0.0f)
                r = pp_follow(p, s.b, s.h, s.span.step(s.off + i) * kPpKeys, s.seq.len, &sm.unit[w], &sm.high[w]);
            const __half2 rel[2] = {__float2half2_rn(r.x), __float2half2_rn(r.y)};
            if (w == 0 && lane == 0) sc.vref = sm.unit[0];
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.sc_full[tile % kPpScales]);
            if (!(ok = pp_wait_warp(&sm.k_empty[st], (use & 1) ^ 1, sm, p))) break;
            pp_store_tile<false>(sm.k[st], kr, w, lane, rel);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.k_full[st]);
            if (i + 1 < s.n) {
                if (((i + 1) & 15) == 0) {
                    fetch(i + 1);
                    vs /= sm.unit[w];  // (of no use where the tiles have their own)
                }
                place(i + 1);
                load(p.c.k, kr);
            }
            if (!(ok = pp_wait_warp(&sm.v_empty[st], (use & 1) ^ 1, sm, p))) break;
            pp_store_tile<true>(sm.v[st], vr, w, lane, rel);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.v_full[st]);
            if (i + 1 < s.n) load(p.c.v, vr);
        }
        u += s.n;
    }
}

// ---- warps 12, 13: the products of row tile 0, 1 ------------------------------------------------
// The whole warp walks the loops with values that the compiler can see to be uniform, and one
// elected lane issues.
__device__ __forceinline__ bool pp_elect() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
__device__ void pp_products(const PaParams &p, PpShared &sm, int u0, int u1) {
    const int lane = threadIdx.x & 31, i = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5) - kPpMmaWarp, 0);
    const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
    const uint32_t ts = tmem + kColS + 128 * i, to = tmem + kColO + 128 * i;
    // K-major operands: 16-byte K slices kPpSlice apart, 8-row groups 128 apart; V (MN-major): 8-key
    // groups 128 apart, 8-column groups kPpSlice apart
    const uint32_t q = pp_desc_lo(smem_u32(sm.q[i]), kPpSlice);
    const uint32_t k0 = pp_desc_lo(smem_u32(sm.k[0]), kPpSlice), v0 = pp_desc_lo(smem_u32(sm.v[0]), 128);
    // half h of a tile: its 64 keys' scores, columns [64 h, 64 h + 64) of the row tile's S
    auto scores = [&](int st, int h) {
        const uint32_t b = k0 + st * (kPpTile >> 4) + h * (8 * 128 >> 4);
        if (pp_elect()) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                pp_mma_ss(ts + 64 * h, q + (k * 2 * kPpSlice >> 4), pp_desc_hi(128), b + (k * 2 * kPpSlice >> 4),
                          pp_desc_hi(128), kPpIdescS, k > 0);
            tc_commit(&sm.s_full[i][h]);
            if (h) tc_commit(&sm.k_empty[st]);
        }
        __syncwarp();
    };
    auto values = [&](int st, int h, bool first) {
        const uint32_t b = v0 + st * (kPpTile >> 4) + h * (4 * 256 >> 4);
        if (pp_elect()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                pp_mma_ts(to, ts + 64 * h + 8 * k, b + (k * 256 >> 4), pp_desc_hi(kPpSlice), kPpIdescV, !(first && k == 0));
            tc_commit(&sm.o_done[i][h]);
            if (h) tc_commit(&sm.v_empty[st]);
        }
        __syncwarp();
    };
    bool ok = true;
    auto wait = [&](uint64_t *bar, int use) {
        ok = ok && pp_wait_warp(bar, (uint32_t)use & 1, sm, p);
        return ok;
    };
    auto test = [&](uint64_t *bar, int use) { return mbar_test_wait(bar, (uint32_t)use & 1); };
    int tile = 0, pieces = 0, used = 0;  // tiles of the CTA so far; pieces and tiles of this row tile
    PpSeg s;
#pragma unroll 1
    for (int u = u0; ok && u < u1;) {
        if (u == u0) pp_seek(p, sm, u, u1, lane, s);
        else pp_next(p, sm, u, u1, lane, s);
        const int n = __shfl_sync(0xffffffffu, s.n, 0);
        if (i == 0 || s.rows > 128) {
            wait(&sm.k_full[tile % kPpStages], tile / kPpStages);
            wait(&sm.q_full[i], pieces);
            tc_fence_after();
            if (ok) scores(tile % kPpStages, 0);
            if (ok) scores(tile % kPpStages, 1);
            // A test of a barrier comes back late (it queues behind the softmaxes' exponentials), so all
            // are asked together and only a phase found open is waited for.
#pragma unroll 1
            for (int y = 0; ok && y < 2 * n; ++y) {
                const int j = y >> 1, h = y & 1, at = tile + j, st = at % kPpStages, next = (at + 1) % kPpStages;
                const bool more = j + 1 < n;
                const bool v_in = test(&sm.v_full[st], at / kPpStages);
                const bool k_in = !more || test(&sm.k_full[next], (at + 1) / kPpStages);
                const bool p_in = test(&sm.p_full[i][h], used + j);
                if (!__all_sync(0xffffffffu, v_in && k_in && p_in)) {
                    wait(&sm.v_full[st], at / kPpStages);
                    if (more) wait(&sm.k_full[next], (at + 1) / kPpStages);
                    if (!wait(&sm.p_full[i][h], used + j)) break;
                }
                tc_fence_after();
                values(st, h, y == 0);
                // the products end in the order of their issue: P is read before the scores of the next
                // tile's half overwrite it
                if (more) scores(next, h);
            }
            ++pieces;
            used += n;
        } else {  // an item of one row tile: this warp's share of the operands' release
#pragma unroll 1
            for (int j = 0; ok && j < n; ++j) {
                const int at = tile + j, st = at % kPpStages;
                if (wait(&sm.k_full[st], at / kPpStages) && lane == 0) mbar_arrive(&sm.k_empty[st]);
                if (wait(&sm.v_full[st], at / kPpStages) && lane == 0) mbar_arrive(&sm.v_empty[st]);
            }
        }
        tile += n;
        u += n;
    }
    if (pp_elect()) tc_commit(&sm.mdone[i]);  // every product has ended before the tensor memory goes
    __syncwarp();
    mbar_wait_bounded(&sm.mdone[i], 0, globaltimer_ns() + kPaTimeoutNs);
    __syncwarp();
}

// ---- warps 0-7: softmax and epilogue ----------------------------------------------------------
// A warp's 32 rows of queries, from row r0 of the sequence's on (none past `last`), to the tile's rows
// from row0 on; the factor of the row of this lane.  A lane takes row lane & 7 of each group of eight
// and 16-byte pieces (lane >> 3) + 4 i: a read covers 64 bytes of eight rows, a write every bank once.
template <typename T>
__device__ __forceinline__ float pp_load_q(const PaParams &p, const PpSeg &s, int r0, int last, uint8_t *tile, int row0) {
    const int lane = threadIdx.x & 31;
    const uint32_t sign = p.scale_log2 < 0.0f ? 0x80008000u : 0u;  // the columns' factors stay >= 0
    uint4 f[4][4];
    float up = 1.0f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int r = r0 + 8 * g + (lane & 7);
        const T *q = static_cast<const T *>(p.q) + (long)(s.seq.row0 + r / p.group) * p.q_stride +
                     (s.h * p.group + r % p.group) * kPgDim + 8 * (lane >> 3);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            f[g][i] = r <= last ? *reinterpret_cast<const uint4 *>(q + 32 * i) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        uint32_t *w = reinterpret_cast<uint32_t *>(f[g]);
        if constexpr (!__is_same(T, __half)) {
            // to f16 with the row's largest value moved to [2^14, 2^15): exact down to 2^-31 of it (f16's
            // subnormals round eight bits from there on), 0 below 2^-39
            float amax = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 8));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 16));
            const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127 - 14, -120), 120);
            const float down = __uint_as_float((uint32_t)(127 - e) << 23);
            if (g == lane >> 3) up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                w[i] = pg_pack2(__uint_as_float(w[i] << 16) * down, __uint_as_float(w[i] & 0xffff0000u) * down,
                                (const __half *)nullptr);
        }
        uint8_t *at = tile + ((row0 >> 3) + g) * 128 + (lane & 7) * 16 + (lane >> 3) * kPpSlice;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4 *>(at + 4 * i * kPpSlice) =
                make_uint4(f[g][i].x ^ sign, f[g][i].y ^ sign, f[g][i].z ^ sign, f[g][i].w ^ sign);
    }
    return up * fabsf(p.scale_log2);
}

template <typename T>
__device__ __forceinline__ void pp_write8(T *out, const float *o, float f) {
    *reinterpret_cast<uint4 *>(out) =
        make_uint4(pg_pack2(o[0] * f, o[1] * f, out), pg_pack2(o[2] * f, o[3] * f, out), pg_pack2(o[4] * f, o[5] * f, out),
                   pg_pack2(o[6] * f, o[7] * f, out));
}

constexpr size_t kPpSlotFloats = (size_t)kPpRows * (kPgDim + 2);

template <typename T>
__device__ void pp_softmax(const PaParams &p, PpShared &sm, int u0, int u1, int share) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = warp >> 2;
    const int row = (warp & 3) * 32 + lane;  // row of the tile, and lane of the tensor memory
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = sm.tmem + lanes + kColS + 128 * i, to = sm.tmem + lanes + kColO + 128 * i;
    int tile = 0, used = 0;
    bool ok = true;  // after a failed wait only the barriers among these warps go on
    float factor = 0.0f;
    // a piece's queries
    auto queries = [&](const PpSeg &s) {
        if (i == 1 && s.rows <= 128) return;
        factor = pp_load_q<T>(p, s, s.row0 + i * 128 + row - lane, s.row0 + s.rows - 1, sm.q[i], row - lane);
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_full[i]);
    };
    PpSeg s;
    pp_seek(p, sm, u0, u1, lane, s);
    queries(s);
#pragma unroll 1
    for (int u = u0; u < u1;) {
        const int end = u - s.off + s.nb, c0 = (u - s.off) / share, c1 = (end - 1) / share;
        float *slot = p.partials + ((size_t)blockIdx.x * 2 + ((int)blockIdx.x == c0 ? 1 : 0)) * kPpSlotFloats;
        const bool mine = i == 0 || s.rows > 128;
        const int r = i * 128 + row;  // of the item
        const bool live = r < s.rows, warp_live = i * 128 + (warp & 3) * 32 < s.rows;
        const int pos = live ? s.seq.pos0 + (s.row0 + r) / p.group : -1;
        float m = -INFINITY, l = 0.0f, vref = 1.0f;
        if (ok && mine) {
#pragma unroll 1
            for (int y = 0; y < 2 * s.n; ++y) {
                const int j = y >> 1, h = y & 1, at = tile + j;
                const PpScale &sc = sm.sc[at % kPpScales];
                const uint32_t tsh = ts + 64 * h;
                // the scales were written before the products of this tile were issued: both tests in one go
                uint64_t *sc_bar = &sm.sc_full[at % kPpScales];
                const bool there = mbar_test_wait(sc_bar, (uint32_t)(at / kPpScales) & 1);
                ok = pp_wait_warp(&sm.s_full[i][h], (uint32_t)(used + j) & 1, sm, p);
                if (!__all_sync(0xffffffffu, there)) ok = ok && pp_wait_warp(sc_bar, (uint32_t)(at / kPpScales) & 1, sm, p);
                if (!ok) break;
                tc_fence_after();
                if (warp_live) {
                    float v[2][32];
                    pp_ld32(tsh, v[0]);
                    pp_ld32(tsh + 32, v[1]);
                    float4 ks = *reinterpret_cast<const float4 *>(sc.k + 4 * h);
                    const float unit = sc.vref;
                    const int key0 = s.span.step(s.off + j) * kPpKeys + 64 * h;
                    const bool whole = key0 + 63 <= pos &&
                                       (p.window <= 0 || pos - key0 < p.window || key0 + 64 <= p.sinks) &
                                           !(fminf(fminf(ks.x, ks.y), fminf(ks.z, ks.w)) < 0.0f);
                    pp_wait_ld(v[0]);
                    pp_hold32(v[1]);
                    bool any = true;
                    if (!__all_sync(0xffffffffu, whole)) {
                        const uint64_t see = pp_sees(pos - key0, p.window, p.sinks - key0, ks);
                        any = __any_sync(0xffffffffu, see != 0);
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const uint32_t bits = (uint32_t)(see >> 32 * c);
#pragma unroll
                            for (int x = 0; x < 32; ++x) v[c][x] = bits >> x & 1 ? v[c][x] : -INFINITY;
                        }
                    }
                    if (any) {
                    // a column's factor: never 0, so that a masked score's -infinity stays one
                    const float col[4] = {fmaxf(ks.x * factor, 1e-35f), fmaxf(ks.y * factor, 1e-35f),
                                          fmaxf(ks.z * factor, 1e-35f), fmaxf(ks.w * factor, 1e-35f)};
                    float top = -INFINITY;
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const float *x = &v[g >> 1][16 * (g & 1)];
                        float mx = x[0], my = x[8];
#pragma unroll
                        for (int c = 1; c < 8; ++c) mx = fmaxf(mx, x[c]), my = fmaxf(my, x[8 + c]);
                        top = fmaxf(top, fmaxf(mx, my) * col[g]);
                    }
                    if (m == -INFINITY) m = top, vref = unit;  // (O and l are zero: there is nothing to scale)
                    if (__any_sync(0xffffffffu, top > m + kPpLazy || unit != vref)) {
                        const float now = fmaxf(m, top), f = now == -INFINITY ? 1.0f : pa_exp2(m - now);
                        m = now;
                        l *= f;
                        if (!(ok = pp_wait_warp(&sm.o_done[i][h ^ 1], (uint32_t)(used + ((y - 1) >> 1)) & 1, sm, p))) break;
                        tc_fence_after();
                        pp_scale_o(to, f * fminf(vref / unit, 0x1p100f));  // (more than 1 / kPpDown only while O is zero)
                        vref = unit;
                    }
                    const float base = m == -INFINITY ? 0.0f : m;
                    const uint64_t less = pp_pair(-base, -base);
                    uint64_t sum = 0;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float(&x)[32] = v[c];
                        uint32_t w[16];
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            const uint64_t col2 = pp_pair(col[2 * c + g], col[2 * c + g]);
#pragma unroll
                            for (int z = 16 * g; z < 16 * g + 16; z += 2) {
                                float e0, e1;
                                uint64_t e = pp_fma2(pp_pair(x[z], x[z + 1]), col2, less);
                                if (z % 8 == 6) {
                                    e = pp_exp2_fma(e);
                                    pp_split(e, e0, e1);
                                } else {
                                    pp_split(e, e0, e1);
                                    e0 = pa_exp2(e0), e1 = pa_exp2(e1);
                                    e = pp_pair(e0, e1);
                                }
                                sum = pp_add2(sum, e);
                                w[z / 2] = pg_pack2(e0, e1, (const __half *)nullptr);
                            }
                        }
                        pp_st16(tsh + 16 * c, w);  // this half of S has been read
                    }
                    float s0, s1;
                    pp_split(sum, s0, s1);
                    l += s0 + s1;
                    } else {  // no row of the warp sees any of it
                        const uint32_t zero[16] = {};
                        pp_st16(tsh, zero);
                        pp_st16(tsh + 16, zero);
                    }
                    pp_wait_st();
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.p_full[i][h]);
            }
        }
        // The next piece's queries, so that its first scores are under way while this one's O is read: the
        // scores that used these queries have all been here.  (After a failed wait the walk goes on, too: all
        // warps reach the barriers of the same cut items.)
        PpSeg next = s;
        if (u + s.n < u1) {
            pp_next(p, sm, u + s.n, u1, lane, next);
            if (ok) queries(next);
        }
        if (ok && mine) {
            ok = pp_wait_warp(&sm.o_done[i][1], (uint32_t)(used + s.n - 1) & 1, sm, p);
            tc_fence_after();
            used += s.n;
            if (ok && warp_live) {
                const long dst = (long)(s.seq.row0 + (s.row0 + r) / p.group) * p.query_heads + s.h * p.group +
                                 (s.row0 + r) % p.group;
                const bool none = m == -INFINITY && l == l;  // the row saw nothing (a NaN score leaves l NaN)
                const float f = c0 != c1 ? vref : none ? 0.0f : vref / l;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    float v[32];
                    pp_ld32(to + 32 * c, v);
                    pp_wait_ld(v);
                    if (live && c0 == c1) {
                        T *out = static_cast<T *>(p.out) + dst * kPgDim + 32 * c;
#pragma unroll
                        for (int x = 0; x < 32; x += 8) pp_write8(out + x, v + x, f);
                    } else if (live) {
                        float4 *out = reinterpret_cast<float4 *>(slot + (size_t)r * kPgDim + 32 * c);
#pragma unroll
                        for (int x = 0; x < 8; ++x)
                            out[x] = make_float4(v[4 * x] * f, v[4 * x + 1] * f, v[4 * x + 2] * f, v[4 * x + 3] * f);
                    }
                }
                if (live && c0 == c1) {
                    if (p.lse) p.lse[dst] = none ? -INFINITY : (m + log2f(l)) * kPaLn2;
                } else if (live) {
                    slot[(size_t)kPpRows * kPgDim + r] = m;
                    slot[(size_t)kPpRows * (kPgDim + 1) + r] = l;
                }
            }
            tc_fence_before();
        }
        if (c0 != c1) {
            named_sync(1, 256);
            if (threadIdx.x == 0) {
                __threadfence();
                // (a block that gave up counts, too: the last one puts the counter back to zero, and the status says
                // that the rows are incomplete)
                sm.last = atomicAdd(p.counters + c0, 1u) == (uint32_t)(c1 - c0);
                __threadfence();
            }
            named_sync(1, 256);
            if (sm.last) {
                // a row's maximum and sum by one thread, then eight rows a warp at a time, their reads in
                // flight together
                auto part = [&](int c) { return p.partials + ((size_t)c * 2 + (c == c0 ? 1 : 0)) * kPpSlotFloats; };
                auto where = [&](int r) {
                    return (long)(s.seq.row0 + (s.row0 + r) / p.group) * p.query_heads + s.h * p.group + (s.row0 + r) % p.group;
                };
                if ((int)threadIdx.x < s.rows) {
                    const int r = threadIdx.x;
                    float top = -INFINITY, l = 0.0f;
#pragma unroll 4
                    for (int c = c0; c <= c1; ++c) top = fmaxf(top, __ldcg(part(c) + (size_t)kPpRows * kPgDim + r));
#pragma unroll 4
                    for (int c = c0; c <= c1; ++c) {
                        const float *a = part(c) + (size_t)kPpRows * kPgDim + r;
                        l += (top == -INFINITY ? 1.0f : pa_exp2(__ldcg(a) - top)) * __ldcg(a + kPpRows);
                    }
                    const bool none = top == -INFINITY && l == l;
                    sm.row_top[r] = top, sm.row_inv[r] = none ? 0.0f : 1.0f / l;
                    if (p.lse) p.lse[where(r)] = none ? -INFINITY : (top + log2f(l)) * kPaLn2;
                }
                named_sync(1, 256);
                constexpr int kAt = 8;
#pragma unroll 1
                for (int r0 = warp * kAt; r0 < s.rows; r0 += 8 * kAt) {
                    float4 acc[kAt];
#pragma unroll
                    for (int x = 0; x < kAt; ++x) acc[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
                    for (int c = c0; c <= c1; ++c) {
                        const float *a = part(c);
                        float4 v[kAt];
                        float f[kAt];
#pragma unroll
                        for (int x = 0; x < kAt; ++x) {
                            const int r = min(r0 + x, s.rows - 1);
                            v[x] = __ldcg(reinterpret_cast<const float4 *>(a + (size_t)r * kPgDim) + lane);
                            f[x] = __ldcg(a + (size_t)kPpRows * kPgDim + r);
                        }
#pragma unroll
                        for (int x = 0; x < kAt; ++x) {
                            const float top = sm.row_top[min(r0 + x, s.rows - 1)];
                            const float g = top == -INFINITY ? 1.0f : pa_exp2(f[x] - top);
                            acc[x].x += g * v[x].x, acc[x].y += g * v[x].y, acc[x].z += g * v[x].z, acc[x].w += g * v[x].w;
                        }
                    }
#pragma unroll
                    for (int x = 0; x < kAt; ++x) {
                        if (r0 + x >= s.rows) break;
                        const float inv = sm.row_inv[r0 + x];
                        T *out = static_cast<T *>(p.out) + where(r0 + x) * kPgDim;
                        reinterpret_cast<uint2 *>(out)[lane] =
                            make_uint2(pg_pack2(acc[x].x * inv, acc[x].y * inv, out),
                                       pg_pack2(acc[x].z * inv, acc[x].w * inv, out));
                    }
                }
                if (threadIdx.x == 0) p.counters[c0] = 0u;
            }
        }
        tile += s.n;
        u += s.n;
        s = next;
    }
}

template <typename T>
__global__ void __launch_bounds__(kPpThreads, 1) paged_attend_prompt_kernel(const __grid_constant__ PaParams p) {
    extern __shared__ uint8_t raw[];
    PpShared &sm = *reinterpret_cast<PpShared *>(raw + ((128u - (smem_u32(raw) & 127u)) & 127u));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.q_full[i], 4);
            for (int h = 0; h < 2; ++h)
                mbar_init(&sm.s_full[i][h], 1), mbar_init(&sm.p_full[i][h], 4), mbar_init(&sm.o_done[i][h], 1);
        }
        for (int i = 0; i < kPpStages; ++i) {
            mbar_init(&sm.k_full[i], 4), mbar_init(&sm.v_full[i], 4);
            mbar_init(&sm.k_empty[i], 2), mbar_init(&sm.v_empty[i], 2);
        }
        for (int i = 0; i < kPpScales; ++i) mbar_init(&sm.sc_full[i], 4);
        mbar_init(&sm.mdone[0], 1), mbar_init(&sm.mdone[1], 1);
        sm.abort = 0;
        fence_mbar_init();
    }
#pragma unroll 1
    for (int b = warp; b < p.b.num_seqs; b += kPpThreads / 32) {
        const int n = pp_seq_units(p, pg_seq(p.b, p.c.page_size, b), lane) * p.c.kv_heads;
        if (lane == 0) sm.prefix[b + 1] = n;
    }
    __syncthreads();
    if (warp == 0) {
        int before = 0;
        if (lane == 0) sm.prefix[0] = 0;
#pragma unroll 1
        for (int b = 0; b < p.b.num_seqs; b += 32) {
            int incl = b + lane < p.b.num_seqs ? sm.prefix[b + lane + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += up;
            }
            if (b + lane < p.b.num_seqs) sm.prefix[b + lane + 1] = before + incl;
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    __syncthreads();
    const int total = sm.prefix[p.b.num_seqs];
    const int share = max((total + (int)gridDim.x - 1) / (int)gridDim.x, 1);
    const int u0 = (int)min((long)share * blockIdx.x, (long)total), u1 = min(u0 + share, total);
    if (u0 >= u1) return;
    if (warp == kPpMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // launched with 128 registers a thread: 256 x 144 + 128 x 136 + 128 x 88 = 512 x 128 (an increase waits for the last
    // group's decrease; a decrease may not name more than the launch gave).  With 152 / 128 / 80 the f16 kernel spills
    // as well and windowed prompts take 165 us instead of 160, a prompt of 4096 at 16384 1460 instead of 1447.
    if (warp < kPpConvWarp0) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
        pp_softmax<T>(p, sm, u0, u1, share);
    } else if (warp < kPpMmaWarp) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
        pp_convert(p, sm, u0, u1);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp < kPpMmaWarp + 2) pp_products(p, sm, u0, u1);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kPpMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sm.tmem), "r"(512));
    }
}

template <typename T>
int pp_launch(const PaParams &p, cudaStream_t s) {
    static std::once_flag once[64];
    static cudaError_t set_rc[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return MMRS_ERR_LAUNCH;
    std::call_once(once[dev], [dev] {
        set_rc[dev] = cudaFuncSetAttribute(paged_attend_prompt_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)kPpSmem);
    });
    if (set_rc[dev] != cudaSuccess) return MMRS_ERR_LAUNCH;
    paged_attend_prompt_kernel<T><<<pa_sm_count(), kPpThreads, kPpSmem, s>>>(p);
    return cudaGetLastError() == cudaSuccess ? MMRS_OK : MMRS_ERR_LAUNCH;
}

}  // namespace

int pa_launch_prompt(const PaParams &p, int type, cudaStream_t s) {
    return type == MMRS_TYPE_F16 ? pp_launch<__half>(p, s) : pp_launch<__nv_bfloat16>(p, s);
}

}  // namespace mmrs
