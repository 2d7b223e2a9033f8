// Shared pieces of the paged-cache kernels: the argument blocks, 16- and 32-bit element access and
// the geometry of a sequence's new tokens.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <stddef.h>

#include "../../include/minimax_paged.h"
#include "common.cuh"

namespace mmrs {

constexpr int kPgDim = MMRS_PAGED_HEAD_DIM;

// Launches a kernel that may start while the one before it in the stream ends: its own launch and
// the setting up of barriers are then out of the way (one token over 4096 positions, call after call:
// 13.3 -> 11.7 us; 48 windowed tokens 26.7 -> 24.7).  Each of these kernels waits (grid_dependency_wait)
// before it touches global memory.  The prompt kernel is launched plainly: with this it was slower
// (windowed prompts 165 -> 173 us).
template <typename... P>
int pg_launch(void (*kernel)(P...), unsigned grid, int threads, size_t smem, cudaStream_t s, const P &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? MMRS_OK : MMRS_ERR_LAUNCH;
}

// Element access by type: four (or eight) consecutive elements as f32.
__device__ __forceinline__ void pg_load4(const float *p, float (&x)[4]) {
    const float4 v = *reinterpret_cast<const float4 *>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
__device__ __forceinline__ void pg_load4(const __half *p, float (&x)[4]) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
__device__ __forceinline__ void pg_load4(const __nv_bfloat16 *p, float (&x)[4]) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pg_pack2(float a, float b, const __half *) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pg_pack2(float a, float b, const __nv_bfloat16 *) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float pg_to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float pg_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float pg_to_float(float v) { return v; }

// Two e4m3 codes (low 16 bits) as two halves, exactly.
__device__ __forceinline__ uint32_t pg_e4m3x2_to_half2(uint32_t two) {
    uint32_t h;
    asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(h) : "r"(two));
    return h;
}

// Four codes as two pairs of halves.
__device__ __forceinline__ void pg_e4m3x4_to_half2(uint32_t four, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(four));
}

// A sequence's new tokens as the kernels see them (cut to the call's bounds): rows
// [row0, row0 + count) of the call, at positions [pos0, pos0 + count), of a length of `len`.
struct PgSeq {
    int row0, count, pos0, len;
};
__device__ __forceinline__ PgSeq pg_seq(const MmrsPagedBatch &b, int page_size, int s) {
    PgSeq q;
    q.row0 = b.cu_q[s];
    int end = b.cu_q[s + 1];
    end = end < b.total_q ? end : b.total_q;
    q.row0 = q.row0 > 0 ? q.row0 : 0;
    q.count = end - q.row0;
    q.count = q.count < 0 ? 0 : q.count > b.max_q ? b.max_q : q.count;
    const long cap = (long)b.table_stride * page_size;
    int len = b.seq_len[s];
    len = len < b.max_len ? len : b.max_len;
    q.len = len < 0 ? 0 : (long)len < cap ? len : (int)cap;
    q.pos0 = q.len - q.count;  // negative when the caller's lengths disagree: those rows see nothing
    return q;
}

int pg_validate(const MmrsPagedCache *c, const MmrsPagedBatch *b);

}  // namespace mmrs
