// Attention of new tokens over a paged e4m3 cache (mmrs_paged_attend): argument checks, workspace, and
// the choice between the two kernels (paged_attend_decode.cu: few rows a KV head, bound by HBM;
// paged_attend_prompt.cu: many, bound by arithmetic; a call that may hold both runs both, each over its
// sequences).
#include <cuda_runtime.h>

#include <mutex>

#include "paged_attend.cuh"

namespace mmrs {
namespace {

// Workspace: a status word, a counter and two partial results (rows of 128 sums, their maximum and
// sum) per CTA.
struct PaLayout {
    size_t counters, partials, total;
};
PaLayout pa_layout(int max_rows) {
    const size_t sms = pa_sm_count(), rows = max_rows <= kPaFewRows ? kPaDecodeRows : 256;
    PaLayout l;
    l.counters = 256;
    l.partials = l.counters + (sizeof(uint32_t) * sms + 255) / 256 * 256;
    l.total = l.partials + sizeof(float) * rows * (kPgDim + 2) * 2 * sms;
    return l;
}
// Rows of a KV head that one sequence can bring when only the batch's total is known.
int pa_rows(long tokens, int group) { return (int)(tokens * group > 256 ? 256 : tokens * group); }

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
    return pa_layout(pa_rows(total_q, query_heads / kv_heads)).total;
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
        workspace_bytes < pa_layout(pa_rows(batch->max_q < batch->total_q ? batch->max_q : batch->total_q,
                                             query_heads / cache->kv_heads)).total)
        return MMRS_ERR_ARG;
    PaParams p = {};
    p.c = *cache;
    p.b = *batch;
    p.q = q, p.out = out, p.lse = lse;
    p.q_stride = q_stride;
    p.query_heads = query_heads, p.group = query_heads / cache->kv_heads;
    p.window = window, p.sinks = sinks;
    p.scale_log2 = scale * kPaLog2e;
    const PaLayout l = pa_layout(kPaDecodeRows);  // (the partial results begin alike in both layouts)
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    p.status = reinterpret_cast<uint32_t *>(ws);
    p.counters = reinterpret_cast<uint32_t *>(ws + l.counters);
    p.partials = reinterpret_cast<float *>(ws + l.partials);
    // a sequence has no more rows than the call; the lengths themselves are on the device
    const long max_q = batch->max_q < batch->total_q ? batch->max_q : batch->total_q;
    const long most = max_q * p.group, few = most < kPaFewRows ? most : kPaFewRows;
    p.b.max_q = (int)max_q;
    p.mixed = most > kPaFewRows;
    p.few_rows = p.mixed && batch->num_seqs == 1 ? 0 : kPaFewRows;  // (one sequence: one kernel, whatever it brings)
    // work units are counted with 32 bits
    if ((long)batch->num_seqs * cache->kv_heads * (few / 8 + 1) * (batch->max_len / 32 + 32) > 0x3fffffffL ||
        ((long)batch->total_q * p.group / 256 + batch->num_seqs) * cache->kv_heads * (batch->max_len / 128 + 1) > 0x3fffffffL)
        return MMRS_ERR_UNSUPPORTED;
    if (p.mixed) {
        const int rc2 = pa_launch_prompt(p, type, (cudaStream_t)stream);
        if (rc2 != MMRS_OK || p.few_rows == 0) return rc2;
    }
    CUtensorMap kmap, vmap;
    const int rows = cache->page_size < 32 ? 16 : 32;
    int mc = pa_make_map(&kmap, cache->k, *cache, rows);
    if (mc == MMRS_OK) mc = pa_make_map(&vmap, cache->v, *cache, rows);
    if (mc != MMRS_OK) return mc;
    return pa_launch_decode(p, kmap, vmap, type, (cudaStream_t)stream);
}
