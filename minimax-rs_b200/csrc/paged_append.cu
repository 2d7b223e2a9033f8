// Appending the new tokens of several sequences to a paged e4m3 cache, the rotary embedding applied
// on the way (mmrs_paged_append).
//
// Rotation (partial rope, pairs (i, i + rope_dim / 2)): (a, b) -> (a c - b s, b c + a s) in f32, each
// product and sum rounded once.  Quantisation: one scale per page and head, the smallest power of
// two with |x| <= 448 scale (448 = 1.75 * 2^8, the largest e4m3 value).  With powers of two a code
// is x's own mantissa rounded to three bits, and a later, larger scale moves only the exponent:
// rounding a page's older codes again changes nothing but e4m3 subnormals.
//
// Bound by HBM at prompt sizes and by a chain of dependent reads (lengths, page, scale, codes) for a
// few tokens.  One launch: blocks of one (page run, KV head) first, then blocks of one token's
// queries, whose reads are under way before the token's sequence and angle are looked up.  A run's
// tokens are looked at twice (largest value, then codes): the first two of each warp stay in
// registers, the others come from L2 again, which was faster than holding them all (128 registers,
// 124-273 us) or none (129 us): 12390 tokens of f32, 48 + 8 heads, 587 MB in 107 us (5.5 TB/s).
#include "paged.cuh"
#include "tma.cuh"

namespace mmrs {
namespace {

constexpr int kApThreads = 128;
constexpr int kApWarps = kApThreads / 32;
constexpr int kApResident = 8;  // blocks an SM: 64 registers
constexpr int kApHeld = 2;  // tokens that a warp keeps in registers between the two looks at them
constexpr float kApMinScale = 5.421010862427522e-20f;  // 2^-64

struct ApParams {
    MmrsPagedCache c;
    MmrsPagedBatch b;
    const void *q, *k, *v;
    long q_stride, k_stride, v_stride;
    int query_heads;
    const float *cos, *sin;
    int rope_dim, rope_positions;
    void *q_out;
    int kv_units;  // page runs (an upper bound) times KV heads; the CTAs after them rotate queries
};

// A lane's four columns of every head of a token: the angles' cosines and sines, its own for the first
// half of the rotated columns and signed for its partner's.
struct ApAngle {
    float c[4], s[4];  // rotated: x c + y s with y the partner column
};
__device__ __forceinline__ ApAngle ap_angle(const ApParams &p, int col, int pos) {
    ApAngle a;
    const int half = p.rope_dim / 2;
    const long at = (long)pos * half;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = col + i;
        a.c[i] = 1.0f, a.s[i] = 0.0f;
        if (d < p.rope_dim) {
            const bool first = d < half;
            a.c[i] = p.cos[at + (first ? d : d - half)];
            a.s[i] = p.sin[at + (first ? d : d - half)];
            if (first) a.s[i] = -a.s[i];
        }
    }
    return a;
}
// Four columns of a head and their partners.
template <typename T>
__device__ __forceinline__ void ap_load4(const ApParams &p, const T *head, int col, float (&x)[4], float (&y)[4]) {
    pg_load4(head + col, x);
    if (col >= p.rope_dim) return;
    const int half = p.rope_dim / 2;
    if (half % 4 == 0) {  // the partners of four columns lie together
        pg_load4(head + (col < half ? col + half : col - half), y);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = col + i;
            y[i] = d < p.rope_dim ? pg_to_float(head[d < half ? d + half : d - half]) : 0.0f;
        }
    }
}
// Rotated: (a, b) -> (a c - b s, b c + a s), each product and sum rounded once.
__device__ __forceinline__ void ap_rotate4(const ApParams &p, int col, const ApAngle &a, float (&x)[4], const float (&y)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (col + i < p.rope_dim) x[i] = __fadd_rn(__fmul_rn(x[i], a.c[i]), __fmul_rn(y[i], a.s[i]));
}

// Smallest power of two s with amax <= 448 s, at least 2^-64; 0 for 0.
__device__ __forceinline__ float ap_scale(float amax) {
    if (!(amax > 0.0f)) return 0.0f;
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);  // 1.75 = 0x600000
    return e < -64 ? kApMinScale : __uint_as_float((uint32_t)(e + 127) << 23);
}

__device__ __forceinline__ uint32_t ap_codes4(const float (&x)[4], float inv) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(x[0] * inv), "f"(x[1] * inv));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(x[2] * inv), "f"(x[3] * inv));
    return (uint32_t)lo | (uint32_t)hi << 16;
}
__device__ __forceinline__ float ap_inverse(float scale) { return scale > 0.0f ? 1.0f / scale : 0.0f; }

// Finds page run `run` of the batch (runs in order of sequence, then page): the sequence, or -1.
__device__ __forceinline__ int ap_find_run(const ApParams &p, int run, int lane, PgSeq &seq, int &page) {
    int before = 0;
    for (int s0 = 0; s0 < p.b.num_seqs; s0 += 32) {
        PgSeq q = {};
        int n = 0;
        if (s0 + lane < p.b.num_seqs) {
            q = pg_seq(p.b, p.c.page_size, s0 + lane);
            if (q.count > 0 && q.pos0 >= 0) n = (q.len - 1) / p.c.page_size - q.pos0 / p.c.page_size + 1;
        }
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, before + incl > run);
        if (past) {
            const int at = __ffs(past) - 1;
            seq.row0 = __shfl_sync(0xffffffffu, q.row0, at);
            seq.count = __shfl_sync(0xffffffffu, q.count, at);
            seq.pos0 = __shfl_sync(0xffffffffu, q.pos0, at);
            seq.len = __shfl_sync(0xffffffffu, q.len, at);
            page = seq.pos0 / p.c.page_size + run - before - __shfl_sync(0xffffffffu, incl - n, at);
            return s0 + at;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    return -1;
}

template <typename T>
__device__ void ap_store_run(const ApParams &p, int unit) {
    __shared__ float s_max[2][kApWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int head = unit % p.c.kv_heads;
    PgSeq seq;
    int at;
    const int s = ap_find_run(p, unit / p.c.kv_heads, lane, seq, at);
    if (s < 0) return;
    const int pid = p.b.page_table[(long)s * p.b.table_stride + at];
    if (pid < 0 || pid >= p.c.num_pages) return;
    const int ps = p.c.page_size, lo = max(seq.pos0, at * ps), hi = min(seq.len, (at + 1) * ps);
    const int col = lane * 4;
    const T *k = static_cast<const T *>(p.k) + head * kPgDim, *v = static_cast<const T *>(p.v) + head * kPgDim;
    float kmax = 0.0f, vmax = 0.0f;
    auto load = [&](int pos, float (&kx)[4], float (&vx)[4]) {
        const long row = seq.row0 + pos - seq.pos0;
        float y[4];
        pg_load4(v + row * p.v_stride + col, vx);
        ap_load4(p, k + row * p.k_stride, col, kx, y);
        ap_rotate4(p, col, ap_angle(p, col, min(pos, p.rope_positions - 1)), kx, y);
        bool fine = true;
#pragma unroll
        for (int i = 0; i < 4; ++i) fine = fine && isfinite(kx[i]) && isfinite(vx[i]);
        return __all_sync(0xffffffffu, fine) != 0;
    };
    // the first look: the largest values (a warp's first kApHeld tokens stay in registers)
    float kx[kApHeld][4], vx[kApHeld][4];
    uint32_t fine = 0;
    auto most = [&](const float (&x)[4], const float (&y)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) kmax = fmaxf(kmax, fabsf(x[i])), vmax = fmaxf(vmax, fabsf(y[i]));
    };
#pragma unroll
    for (int t = 0; t < kApHeld; ++t) {
        const int pos = lo + warp + t * kApWarps;
        if (pos < hi && load(pos, kx[t], vx[t])) {
            fine |= 1u << t;
            most(kx[t], vx[t]);
        }
    }
    for (int pos = lo + warp + kApHeld * kApWarps; pos < hi; pos += kApWarps) {
        float x[4], y[4];
        if (load(pos, x, y)) most(x, y);
    }
    kmax = warp_max_butterfly(kmax), vmax = warp_max_butterfly(vmax);
    if (lane == 0) s_max[0][warp] = kmax, s_max[1][warp] = vmax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kApWarps; ++w) kmax = fmaxf(kmax, s_max[0][w]), vmax = fmaxf(vmax, s_max[1][w]);
    const long ph = (long)pid * p.c.kv_heads + head;
    float scale[2] = {ap_scale(kmax), ap_scale(vmax)};
    uint8_t *codes[2] = {static_cast<uint8_t *>(p.c.k) + ph * ps * kPgDim,
                         static_cast<uint8_t *>(p.c.v) + ph * ps * kPgDim};
    float *scales[2] = {p.c.k_scale + ph, p.c.v_scale + ph};
    const int older = lo - at * ps;  // slots that earlier calls filled
    if (older > 0) {
        const float was[2] = {*scales[0], *scales[1]};
        __syncthreads();  // all threads have read the scales before thread 0 replaces them
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if (was[t] >= scale[t]) {
                scale[t] = was[t];
                continue;
            }
            const float ratio = was[t] / scale[t];
            for (int i = threadIdx.x; i < older * kPgDim / 4; i += kApThreads) {
                uint32_t *w = reinterpret_cast<uint32_t *>(codes[t]) + i;
                const uint32_t c = *w;
                const uint32_t h0 = pg_e4m3x2_to_half2(c & 0xffffu), h1 = pg_e4m3x2_to_half2(c >> 16);
                const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&h0));
                const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&h1));
                const float x[4] = {a.x, a.y, b.x, b.y};
                *w = ap_codes4(x, ratio);
            }
        }
    }
    if (threadIdx.x == 0) *scales[0] = scale[0], *scales[1] = scale[1];
    const float kinv = ap_inverse(scale[0]), vinv = ap_inverse(scale[1]);
    auto store = [&](int pos, const float (&x)[4], const float (&y)[4], bool ok) {
        const long at4 = ((long)(pos - at * ps) * kPgDim + col) / 4;
        reinterpret_cast<uint32_t *>(codes[0])[at4] = ok ? ap_codes4(x, kinv) : 0x7f7f7f7fu;
        reinterpret_cast<uint32_t *>(codes[1])[at4] = ok ? ap_codes4(y, vinv) : 0u;
    };
#pragma unroll
    for (int t = 0; t < kApHeld; ++t) {
        const int pos = lo + warp + t * kApWarps;
        if (pos < hi) store(pos, kx[t], vx[t], (fine >> t) & 1);
    }
    for (int pos = lo + warp + kApHeld * kApWarps; pos < hi; pos += kApWarps) {
        float x[4], y[4];
        const bool ok = load(pos, x, y);
        store(pos, x, y, ok);
    }
}

template <typename T, typename O>
__device__ void ap_rotate_row(const ApParams &p, int row) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = lane * 4;
    const T *q = static_cast<const T *>(p.q) + (long)row * p.q_stride;
    O *out = static_cast<O *>(p.q_out) + (long)row * p.query_heads * kPgDim;
    // a warp's first heads, under way while the row's sequence is looked up
    constexpr int kAhead = 4;
    float x[kAhead][4], y[kAhead][4];
    auto load = [&](int h0) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (h0 + i * kApWarps < p.query_heads) ap_load4(p, q + (h0 + i * kApWarps) * kPgDim, col, x[i], y[i]);
    };
    load(warp);
    // the row's sequence: how many sequences end at or before it
    int s = 0;
    for (int s0 = 0; s0 < p.b.num_seqs; s0 += 32)
        s += __popc(__ballot_sync(0xffffffffu, s0 + lane < p.b.num_seqs && p.b.cu_q[s0 + lane + 1] <= row));
    if (s >= p.b.num_seqs) return;
    const PgSeq seq = pg_seq(p.b, p.c.page_size, s);
    const int pos = min(max(seq.pos0 + row - seq.row0, 0), p.rope_positions - 1);
    // a lane has the same columns of every head, so one angle serves them all
    const ApAngle angle = ap_angle(p, col, pos);
    for (int h0 = warp; h0 < p.query_heads;) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int h = h0 + i * kApWarps;
            if (h >= p.query_heads) break;
            ap_rotate4(p, col, angle, x[i], y[i]);
            reinterpret_cast<uint2 *>(out + h * kPgDim)[lane] =
                make_uint2(pg_pack2(x[i][0], x[i][1], out), pg_pack2(x[i][2], x[i][3], out));
        }
        h0 += kAhead * kApWarps;
        load(h0);
    }
}

template <typename T, typename O>
__global__ void __launch_bounds__(kApThreads, kApResident) paged_append_kernel(const __grid_constant__ ApParams p) {
    launch_dependents();
    grid_dependency_wait();
    if ((int)blockIdx.x < p.kv_units)
        ap_store_run<T>(p, blockIdx.x);
    else
        ap_rotate_row<T, O>(p, blockIdx.x - p.kv_units);
}

template <typename T, typename O>
int ap_launch(const ApParams &p, cudaStream_t s) {
    const long grid = (long)p.kv_units + (p.q ? p.b.total_q : 0);
    if (grid > 0x7fffffffL) return MMRS_ERR_UNSUPPORTED;
    return pg_launch(paged_append_kernel<T, O>, (unsigned)grid, kApThreads, 0, s, p);
}

}  // namespace

int pg_validate(const MmrsPagedCache *c, const MmrsPagedBatch *b) {
    if (!c || !b || !c->k || !c->v || !c->k_scale || !c->v_scale) return MMRS_ERR_ARG;
    if (((uintptr_t)c->k & 127u) || ((uintptr_t)c->v & 127u)) return MMRS_ERR_ARG;
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        return MMRS_ERR_UNSUPPORTED;
    if (c->num_pages < 1 || c->kv_heads < 1) return MMRS_ERR_ARG;
    // rows of 128 codes are addressed with 32 bits
    if ((long)c->num_pages * c->kv_heads * c->page_size > 0x7fffffffL) return MMRS_ERR_UNSUPPORTED;
    if (b->num_seqs < 0 || b->total_q < 0 || b->max_q < 0 || b->max_len < 0 || b->table_stride < 0) return MMRS_ERR_ARG;
    if (b->num_seqs > MMRS_PAGED_MAX_SEQS) return MMRS_ERR_UNSUPPORTED;
    if (b->num_seqs == 0 || b->total_q == 0) return MMRS_OK;
    if (!b->cu_q || !b->seq_len || !b->page_table) return MMRS_ERR_ARG;
    if (b->max_q < 1 || b->max_len < 1 || (long)b->table_stride * c->page_size < b->max_len) return MMRS_ERR_ARG;
    return MMRS_OK;
}

}  // namespace mmrs

using namespace mmrs;

extern "C" int mmrs_paged_append(const MmrsPagedCache *cache, const MmrsPagedBatch *batch, const void *q, const void *k,
                                 const void *v, int64_t q_stride, int64_t k_stride, int64_t v_stride, int in_type,
                                 int query_heads, const float *rope_cos, const float *rope_sin, int rope_dim,
                                 int rope_positions, void *q_out, int out_type, mmrs_stream_t stream) {
    const int rc = pg_validate(cache, batch);
    if (rc != MMRS_OK) return rc;
    if (in_type < MMRS_TYPE_F32 || in_type > MMRS_TYPE_BF16) return MMRS_ERR_UNSUPPORTED;
    if (rope_dim < 0 || rope_dim > kPgDim || rope_dim % 2) return MMRS_ERR_UNSUPPORTED;
    if ((q == nullptr) != (q_out == nullptr)) return MMRS_ERR_ARG;
    if (batch->num_seqs == 0 || batch->total_q == 0) return MMRS_OK;
    if (!k || !v || (rope_dim && (!rope_cos || !rope_sin || rope_positions < batch->max_len))) return MMRS_ERR_ARG;
    const int align = in_type == MMRS_TYPE_F32 ? 4 : 8;
    if (k_stride < (int64_t)cache->kv_heads * kPgDim || v_stride < (int64_t)cache->kv_heads * kPgDim ||
        k_stride % align || v_stride % align || ((uintptr_t)k & 15u) || ((uintptr_t)v & 15u))
        return MMRS_ERR_ARG;
    if (q) {
        if (out_type != MMRS_TYPE_F16 && out_type != MMRS_TYPE_BF16) return MMRS_ERR_UNSUPPORTED;
        if (query_heads < 1 || q_stride < (int64_t)query_heads * kPgDim || q_stride % align || ((uintptr_t)q & 15u) ||
            ((uintptr_t)q_out & 15u))
            return MMRS_ERR_ARG;
    }
    const long runs = (long)batch->total_q / cache->page_size + 2L * batch->num_seqs;
    const long units = (runs < batch->total_q ? runs : batch->total_q) * cache->kv_heads;
    if (units > 0x3fffffffL) return MMRS_ERR_UNSUPPORTED;
    ApParams p = {};
    p.c = *cache;
    p.b = *batch;
    p.q = q, p.k = k, p.v = v;
    p.q_stride = q_stride, p.k_stride = k_stride, p.v_stride = v_stride;
    p.query_heads = q ? query_heads : 0;
    p.cos = rope_cos, p.sin = rope_sin;
    p.rope_dim = rope_dim, p.rope_positions = rope_dim ? rope_positions : 0x7fffffff;
    p.q_out = q_out;
    p.kv_units = (int)units;
    cudaStream_t s = (cudaStream_t)stream;
    const bool half_out = !q || out_type == MMRS_TYPE_F16;
    if (in_type == MMRS_TYPE_F32) return half_out ? ap_launch<float, __half>(p, s) : ap_launch<float, __nv_bfloat16>(p, s);
    if (in_type == MMRS_TYPE_F16)
        return half_out ? ap_launch<__half, __half>(p, s) : ap_launch<__half, __nv_bfloat16>(p, s);
    return half_out ? ap_launch<__nv_bfloat16, __half>(p, s) : ap_launch<__nv_bfloat16, __nv_bfloat16>(p, s);
}
