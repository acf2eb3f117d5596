// row_utils.cuh — device helpers of the row operators: 16-bit element types,
// vectors of elements, ordered keys, warp and block sums.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "device_utils.cuh"

namespace heph {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v) {
    if constexpr (std::is_same_v<T, float>) return v;
    else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(v);
    else return __float2half_rn(v);
}

// N adjacent elements, moved by one access: of 16 bytes at most, as no operand
// or workspace is known to be aligned to more.
template <typename T, int N> struct alignas(sizeof(T) * N) Pack {
    static_assert(sizeof(T) * N <= 16);
    T e[N];
};

// Calls f.template operator()<T>() with the element type of `dt`.
template <typename F> heph_status dispatch_row_dtype(heph_row_dtype dt, F &&f) {
    switch (dt) {
        case HEPH_ROW_F32: return f.template operator()<float>();
        case HEPH_ROW_BF16: return f.template operator()<__nv_bfloat16>();
        case HEPH_ROW_F16: return f.template operator()<__half>();
        default: return fail(HEPH_INVALID_CONFIGURATION, "unsupported row element type");
    }
}

// An unsigned key in the order of the floats; -0 and +0 have the same key,
// NaN has that of -inf.
__device__ __forceinline__ uint32_t ordered_number(float v) {  // v is not NaN
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint32_t ordered_key(float v) { return ordered_number(v == v ? v : -INFINITY); }
__device__ __forceinline__ float key_value(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ float warp_sum(float v) { return warp_fold<float, OP_SUM>(v); }
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v = fmaxf(v, shfl_xor(v, m));
    return v;
}

// Launches `kernel`; the status is that of this launch alone.
template <typename... P, typename... A>
heph_status launch_rows(const char *what, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                        A &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    HEPH_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, P(args)...), HEPH_DISPATCH_FAILED, what);
    return HEPH_OK;
}

// A kernel that follows another of the same call: its blocks may start before
// that one ends, from its let_next_start() on, and see what it wrote after
// after_previous().
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename... P, typename... A>
heph_status launch_next(const char *what, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                        A &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    HEPH_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, P(args)...), HEPH_DISPATCH_FAILED, what);
    return HEPH_OK;
}

// The same with the blocks in clusters of `cluster`.
template <typename... P, typename... A>
heph_status launch_clusters(const char *what, void (*kernel)(P...), dim3 grid, dim3 block, uint32_t cluster, size_t smem,
                            cudaStream_t stream, A &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    HEPH_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, P(args)...), HEPH_DISPATCH_FAILED, what);
    return HEPH_OK;
}

}  // namespace heph
