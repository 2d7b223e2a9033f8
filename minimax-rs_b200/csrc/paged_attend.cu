// Attention of new tokens over a paged e4m3 cache (mmrs_paged_attend).
//
// One CTA takes 16 rows (new tokens times the query heads of one KV head) of a sequence and walks
// the sequence's positions in tiles of 32 with the running maximum and sum of a softmax.
#include <cuda_runtime.h>

#include <mutex>

#include "paged_attend.cuh"

namespace mmrs {
namespace {

constexpr int kPaThreads = 128;
constexpr int kPaRows = 16;
constexpr int kPaKeys = 32;

template <typename T>
__global__ void __launch_bounds__(kPaThreads) paged_attend_simple_kernel(const __grid_constant__ PaParams p) {
    __shared__ float s_q[kPaRows][kPgDim], s_k[kPaKeys][kPgDim + 1], s_v[kPaKeys][kPgDim], s_p[kPaRows][kPaKeys];
    __shared__ float s_m[kPaRows], s_l[kPaRows], s_fac[kPaRows];
    __shared__ int s_pid[kPaKeys];
    const int tid = threadIdx.x, head = blockIdx.y, s = blockIdx.z;
    const PgSeq seq = pg_seq(p.b, p.c.page_size, s);
    const int row0 = blockIdx.x * kPaRows, rows = min(kPaRows, seq.count * p.group - row0);
    if (rows <= 0) return;
    const T *q = static_cast<const T *>(p.q);
    for (int i = tid; i < rows * kPgDim; i += kPaThreads) {
        const int r = row0 + i / kPgDim, d = i % kPgDim;
        s_q[i / kPgDim][d] = pg_to_float(
            q[(long)(seq.row0 + r / p.group) * p.q_stride + (head * p.group + r % p.group) * kPgDim + d]);
    }
    if (tid < kPaRows) s_m[tid] = -INFINITY, s_l[tid] = 0.0f;
    float o[kPaRows] = {};
    const int last = min(seq.len, seq.pos0 + (row0 + rows - 1) / p.group + 1);
    const int first = p.window > 0 ? max(0, seq.pos0 + row0 / p.group - p.window + 1) : 0;
    const int ps = p.c.page_size;
    for (int j0 = 0; j0 < last; j0 += kPaKeys) {
        if (p.window > 0 && j0 >= p.sinks && j0 + kPaKeys <= first) continue;
        __syncthreads();
        if (tid < kPaKeys) {
            const int j = j0 + tid;
            int pid = j < last ? p.b.page_table[(long)s * p.b.table_stride + j / ps] : -1;
            s_pid[tid] = pid < 0 || pid >= p.c.num_pages ? -1 : pid;
        }
        __syncthreads();
        for (int i = tid; i < kPaKeys * kPgDim; i += kPaThreads) {
            const int key = i / kPgDim, d = i % kPgDim, pid = s_pid[key];
            float kx = 0.0f, vx = 0.0f;
            if (pid >= 0) {
                const long ph = (long)pid * p.c.kv_heads + head, at = (ph * ps + (j0 + key) % ps) * kPgDim + d;
                kx = (float)static_cast<const __nv_fp8_e4m3 *>(p.c.k)[at] * p.c.k_scale[ph];
                vx = (float)static_cast<const __nv_fp8_e4m3 *>(p.c.v)[at] * p.c.v_scale[ph];
            }
            s_k[key][d] = kx;
            s_v[key][d] = vx;
        }
        __syncthreads();
        for (int i = tid; i < kPaRows * kPaKeys; i += kPaThreads) {
            const int r = i / kPaKeys, key = i % kPaKeys, j = j0 + key, pos = seq.pos0 + (row0 + r) / p.group;
            const bool sees = r < rows && s_pid[key] >= 0 && j <= pos && pos >= 0 &&
                              (p.window <= 0 || pos - j < p.window || j < p.sinks);
            float x = -INFINITY;
            if (sees) {
                x = 0.0f;
                for (int d = 0; d < kPgDim; ++d) x = fmaf(s_q[r][d], s_k[key][d], x);
                x *= p.scale_log2 * kPaLn2;
            }
            s_p[r][key] = x;
        }
        __syncthreads();
        if (tid < kPaRows) {
            float m = s_m[tid], sum = 0.0f;
            for (int key = 0; key < kPaKeys; ++key) m = s_p[tid][key] > m || s_p[tid][key] != s_p[tid][key] ? s_p[tid][key] : m;
            for (int key = 0; key < kPaKeys; ++key) {
                const float e = s_p[tid][key] == -INFINITY ? 0.0f : expf(s_p[tid][key] - m);
                s_p[tid][key] = e;
                sum += e;
            }
            const float fac = s_m[tid] == -INFINITY ? 0.0f : expf(s_m[tid] - m);
            s_fac[tid] = fac;
            s_l[tid] = s_l[tid] * fac + sum;
            s_m[tid] = m;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kPaRows; ++r) {
            float acc = o[r] * s_fac[r];
            for (int key = 0; key < kPaKeys; ++key)
                if (s_p[r][key] != 0.0f) acc = fmaf(s_p[r][key], s_v[key][tid], acc);
            o[r] = acc;
        }
    }
    __syncthreads();
    T *out = static_cast<T *>(p.out);
#pragma unroll
    for (int r = 0; r < kPaRows; ++r) {
        if (r >= rows) break;
        const long at = (long)(seq.row0 + (row0 + r) / p.group) * p.query_heads + head * p.group + (row0 + r) % p.group;
        const float l = s_l[r];
        out[at * kPgDim + tid] = (T)(l == 0.0f ? 0.0f : o[r] / l);
        if (p.lse && tid == 0) p.lse[at] = l == 0.0f ? -INFINITY : s_m[r] + logf(l);
    }
}

// Workspace: a status word, one counter per (sequence, KV head), two partial results per CTA.
constexpr size_t kPaSlot = sizeof(float) * 32 * (kPgDim + 2);
struct PaLayout {
    size_t counters, partials, total;
};
PaLayout pa_layout(int num_seqs, int kv_heads) {
    PaLayout l;
    l.counters = 256;
    l.partials = l.counters + (sizeof(uint32_t) * num_seqs * kv_heads + 255) / 256 * 256;
    l.total = l.partials + kPaSlot * 2 * pa_sm_count();
    return l;
}

}  // namespace

int pa_sm_count() {
    static std::once_flag once[64];
    static int sms[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    std::call_once(once[dev], [dev] {
        int n = 0;
        sms[dev] = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0 ? n : 148;
    });
    return sms[dev];
}

int pa_make_map(CUtensorMap *map, const void *codes, const MmrsPagedCache &c, int rows) {
    const auto encode = tensor_map_encoder();
    if (!encode) return MMRS_ERR_LAUNCH;
    const cuuint64_t dims[2] = {(cuuint64_t)kPgDim, (cuuint64_t)c.num_pages * c.kv_heads * c.page_size};
    const cuuint64_t strides[1] = {(cuuint64_t)kPgDim};
    const cuuint32_t box[2] = {(cuuint32_t)kPgDim, (cuuint32_t)rows}, elem[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(codes), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? MMRS_OK
               : MMRS_ERR_LAUNCH;
}

}  // namespace mmrs

using namespace mmrs;

extern "C" size_t mmrs_paged_attend_workspace_bytes(int num_seqs, int total_q, int query_heads, int kv_heads) {
    if (num_seqs < 0 || num_seqs > kPaMaxSeqs || total_q < 0 || kv_heads < 1 || query_heads < kv_heads ||
        query_heads % kv_heads || query_heads / kv_heads > MMRS_PAGED_MAX_GROUP)
        return 0;
    return pa_layout(num_seqs, kv_heads).total;
}

extern "C" int mmrs_paged_attend_status(const void *workspace) {
    if (!workspace) return MMRS_ERR_ARG;
    uint32_t st = 0;
    if (cudaMemcpy(&st, workspace, sizeof(st), cudaMemcpyDeviceToHost) != cudaSuccess) return MMRS_ERR_LAUNCH;
    return (int)st;
}

extern "C" int mmrs_paged_attend(const MmrsPagedCache *cache, const MmrsPagedBatch *batch, const void *q,
                                 int64_t q_stride, int type, int query_heads, float scale, int window, int sinks,
                                 void *out, float *lse, void *workspace, size_t workspace_bytes, mmrs_stream_t stream) {
    const int rc = pg_validate(cache, batch);
    if (rc != MMRS_OK) return rc;
    if (type != MMRS_TYPE_F16 && type != MMRS_TYPE_BF16) return MMRS_ERR_UNSUPPORTED;
    if (query_heads < 1 || query_heads % cache->kv_heads || query_heads / cache->kv_heads > MMRS_PAGED_MAX_GROUP)
        return MMRS_ERR_UNSUPPORTED;
    if (!isfinite(scale) || window < 0 || sinks < 0) return MMRS_ERR_ARG;
    if (batch->num_seqs == 0 || batch->total_q == 0) return MMRS_OK;
    if (!q || !out || ((uintptr_t)q & 15u) || ((uintptr_t)out & 15u) || q_stride % 8 ||
        q_stride < (int64_t)query_heads * kPgDim)
        return MMRS_ERR_ARG;
    if (!workspace || ((uintptr_t)workspace & 255u) ||
        workspace_bytes < pa_layout(batch->num_seqs, cache->kv_heads).total)
        return MMRS_ERR_ARG;
    PaParams p = {};
    p.c = *cache;
    p.b = *batch;
    p.q = q, p.out = out, p.lse = lse;
    p.q_stride = q_stride;
    p.query_heads = query_heads, p.group = query_heads / cache->kv_heads;
    p.window = window, p.sinks = sinks;
    p.scale_log2 = scale * kPaLog2e;
    const PaLayout l = pa_layout(batch->num_seqs, cache->kv_heads);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    p.status = reinterpret_cast<uint32_t *>(ws);
    p.counters = reinterpret_cast<uint32_t *>(ws + l.counters);
    p.partials = reinterpret_cast<float *>(ws + l.partials);
    // units of work (16 positions of a KV head) are counted with 32 bits
    if ((long)batch->num_seqs * cache->kv_heads * ((batch->max_len + 15) / 16) > 0x3fffffffL) return MMRS_ERR_UNSUPPORTED;
    if ((long)batch->max_q * p.group <= 32) {
        CUtensorMap kmap, vmap;
        int mc = pa_make_map(&kmap, cache->k, *cache, 16);
        if (mc == MMRS_OK) mc = pa_make_map(&vmap, cache->v, *cache, 16);
        return mc != MMRS_OK ? mc : pa_launch_decode(p, kmap, vmap, type, (cudaStream_t)stream);
    }
    const long tiles = ((long)batch->max_q * p.group + kPaRows - 1) / kPaRows;
    if (tiles > 0x7fffffffL || cache->kv_heads > 65535) return MMRS_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)tiles, cache->kv_heads, batch->num_seqs);
    if (type == MMRS_TYPE_F16)
        paged_attend_simple_kernel<__half><<<grid, kPaThreads, 0, (cudaStream_t)stream>>>(p);
    else
        paged_attend_simple_kernel<__nv_bfloat16><<<grid, kPaThreads, 0, (cudaStream_t)stream>>>(p);
    return cudaGetLastError() == cudaSuccess ? MMRS_OK : MMRS_ERR_LAUNCH;
}
