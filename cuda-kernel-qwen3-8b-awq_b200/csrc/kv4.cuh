// Paged 4-bit KV cache: layout of a page and the arithmetic of a row, shared by the operators that write and read it.
//
// 16 tokens of one KV head lie together, a tile of 2176 bytes: 16 rows of 64 bytes of K codes (byte i: dim 2i in the low nibble), the same
// of V, 16 pairs (scale, minimum) of K, 16 of V.  A page is [kv_heads][page_size / 16] tiles, so that any part of a page that a
// kernel needs is one contiguous piece, aligned for a bulk copy.  A row stands for code * scale + minimum: one scale for the 128 dims of a
// token and head, which lets attention take it out of its sums.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace qw3 {

constexpr int KV4_TILE_TOKENS = 16;
constexpr int KV4_TILE_BYTES = 2176;
constexpr int KV4_V = 1024, KV4_KP = 2048, KV4_VP = 2112;   // offsets of the V codes and of the pairs of K and V in a tile

constexpr float KV4_MAX_SCALE = 2e38f;   // of scores: times log2(e) it stays in fp32

// Codes of the workspace's error word: an index or a length outside the buffers of the call (QW3_ERR_RANGE).
enum { KV4_ERR_LENGTH = 0xE0001, KV4_ERR_TABLE = 0xE0002, KV4_ERR_PAGES = 0xE0003, KV4_ERR_TOKENS = 0xE0004, KV4_ERR_FREE_ID = 0xE0005,
       KV4_ERR_APPEND_SLOT = 0xE0011, KV4_ERR_APPEND_POS = 0xE0012, KV4_ERR_READ_SLOT = 0xE0021, KV4_ERR_DECODE_PAGE = 0xE0031,
       KV4_ERR_DECODE_LEN = 0xE0032, KV4_ERR_PACKED_CU = 0xE0041 };

const Workspace* ws_struct(qw3_ws_t ws);
bool ws_pdl(qw3_ws_t ws);
// Checks of a pool and a workspace that every operator on them makes; `who` names the entry point.
int kv4_check(const char* who, const Qw3Kv4Pool* pool, qw3_ws_t ws);
int ws_on_device(const char* who, qw3_ws_t ws);

#ifdef __CUDACC__

template <class T> struct RowType;
template <> struct RowType<__half> {
    static constexpr float FLOOR = 5.9604644775390625e-8f;   // 2^-24, the smallest scale that is not zero
    static constexpr float CEIL = 65504.0f;
    static __device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <> struct RowType<__nv_bfloat16> {
    static constexpr float FLOOR = 8.673617379884035e-19f;   // 2^-60 and 2^60: products and quotients of scales stay inside fp32; a row
    static constexpr float CEIL = 1.152921504606846976e18f;  // whose range passes 15 * 2^60 reads back as NaN
    static __device__ __forceinline__ float2 unpack(uint32_t w) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};

// two fp32 operations in one instruction, each rounded to nearest
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(*reinterpret_cast<unsigned long long*>(&r)) : "l"(*reinterpret_cast<const unsigned long long*>(&a)), "l"(*reinterpret_cast<const unsigned long long*>(&b)));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(*reinterpret_cast<unsigned long long*>(&r)) : "l"(*reinterpret_cast<const unsigned long long*>(&a)), "l"(*reinterpret_cast<const unsigned long long*>(&b)));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(*reinterpret_cast<unsigned long long*>(&r)) : "l"(*reinterpret_cast<const unsigned long long*>(&a)), "l"(*reinterpret_cast<const unsigned long long*>(&b)), "l"(*reinterpret_cast<const unsigned long long*>(&c)));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {   // NaN where either is
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// untiled bulk copy global -> shared; addresses and size are multiples of 16
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void kv4_error(int* err, int code) { atomicCAS(err, 0, code); }

// Launch helper: optional programmatic dependent launch and cluster size.
template <typename... KArgs, typename... Args>
cudaError_t kv4_launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool pdl, int cluster, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

#endif

}  // namespace qw3
