// row_norm.cu — root-mean-square norm of rows, with the residual's addition
// and 8-bit output, and its gradient.
//
//   s = x + residual,  rstd = 1 / sqrt(mean(s^2) + eps),  y = w s rstd
//   e4m3 output: scale = max(max|y|, 2^-100) / 448 over a row or a group of
//   columns, q = y / scale.
//   gradient:    dx = rstd w dy - s rstd^3 mean(w dy s) + dsum,
//                dw = sum over rows of dy s rstd
//
// All in 32 bits from the unrounded sum s; each output is rounded once.
#include <cuda_fp8.h>

#include "row_ops.h"
#include "row_utils.cuh"

namespace heph {

namespace {

constexpr float kFp8Max = 448.0f;       // largest finite e4m3 value
constexpr float kFp8Floor = 0x1p-100f;  // smallest maximum a scale is made for: keeps 1 / scale finite

struct NormParams {
    const void *x, *residual, *weight;
    void *y, *sum;
    float *scales;
    int64_t x_stride, residual_stride;
    float eps;
    uint32_t rows, cols;
    uint32_t group, groups;  // columns per scale, scales per row
    bool weight_f32;
};

// V weights from `col` on (all ones without a weight vector).
template <typename T, int V>
__device__ __forceinline__ void load_weight(const void *weight, bool f32, uint32_t col, float (&w)[V]) {
    if (!weight) {
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = 1.0f;
    } else if (f32) {
        constexpr int N = V < 4 ? V : 4;
#pragma unroll
        for (int i = 0; i < V / N; ++i) {
            const auto u = *reinterpret_cast<const Pack<float, N> *>(static_cast<const float *>(weight) + col + i * N);
#pragma unroll
            for (int j = 0; j < N; ++j) w[i * N + j] = u.e[j];
        }
    } else {
        const auto u = *reinterpret_cast<const Pack<T, V> *>(static_cast<const T *>(weight) + col);
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = to_f32(u.e[j]);
    }
}

template <typename T, int V> __device__ __forceinline__ void store_as(T *dst, const float (&v)[V]) {
    Pack<T, V> u;
#pragma unroll
    for (int j = 0; j < V; ++j) u.e[j] = from_f32<T>(v[j]);
    *reinterpret_cast<Pack<T, V> *>(dst) = u;
}

template <int V> __device__ __forceinline__ void store_fp8(void *dst, const float (&v)[V]) {
    if constexpr (V == 1) {
        *static_cast<__nv_fp8_storage_t *>(dst) = __nv_cvt_float_to_fp8(v[0], __NV_SATFINITE, __NV_E4M3);
    } else {
        Pack<__nv_fp8x2_storage_t, V / 2> u;
#pragma unroll
        for (int j = 0; j < V / 2; ++j)
            u.e[j] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * j], v[2 * j + 1]), __NV_SATFINITE, __NV_E4M3);
        *static_cast<Pack<__nv_fp8x2_storage_t, V / 2> *>(dst) = u;
    }
}

// Sum of `a` and (MAX) maximum or (otherwise) sum of `b` over the block, or
// over the warp when rows are warps; every thread gets both.
template <bool MAX> __device__ __forceinline__ void row_fold(float &a, float &b, bool warp_rows, float (*red)[32]) {
    a = warp_sum(a);
    b = MAX ? warp_max(b) : warp_sum(b);
    if (warp_rows || blockDim.x == 32) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (lane == 0) {
        red[0][warp] = a;
        red[1][warp] = b;
    }
    __syncthreads();
    a = warp_sum(lane < warps ? red[0][lane] : 0.0f);
    const float o = lane < warps ? red[1][lane] : 0.0f;
    b = MAX ? warp_max(o) : warp_sum(o);
}

__device__ __forceinline__ float scale_of(float amax) { return fmaxf(amax, kFp8Floor) / kFp8Max; }

// A row (or, blockDim.y > 1, a row per warp) whose C x V values per thread
// stay in registers between the one read and the one write.
template <typename T, int V, int C, bool FP8>
__global__ void __launch_bounds__(1024) norm_kernel(NormParams p) {
    extern __shared__ float group_max[];  // used where a group spans warps
    __shared__ float red[2][32];
    const bool warp_rows = blockDim.y > 1;
    const uint32_t row = blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= p.rows) return;  // whole warps, which no block barrier waits for
    const uint32_t t = threadIdx.x, step = blockDim.x * V;
    const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
    const T *res = p.residual ? static_cast<const T *>(p.residual) + row * p.residual_stride : nullptr;
    const bool by_group = FP8 && p.groups > 1;
    const uint32_t lanes = FP8 ? p.group / V : 0;  // threads that share a scale
    const bool wide_group = by_group && lanes > 32;
    if (wide_group) {
        for (uint32_t g = t; g < p.groups; g += blockDim.x) group_max[g] = 0.0f;
        __syncthreads();
    }

    Pack<T, V> ux[C], ur[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t col = c * step + t * V;
        if (col < p.cols) {
            ux[c] = *reinterpret_cast<const Pack<T, V> *>(x + col);
            if (res) ur[c] = *reinterpret_cast<const Pack<T, V> *>(res + col);
        }
    }
    float v[C][V], ss = 0.0f, amax = 0.0f, gmax[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t col = c * step + t * V;
        gmax[c] = 0.0f;
        if (col < p.cols) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[c][j] = to_f32(ux[c].e[j]);
                if (res) v[c][j] += to_f32(ur[c].e[j]);
                ss += v[c][j] * v[c][j];
            }
            if (res) store_as<T, V>(static_cast<T *>(p.sum) + (int64_t)row * p.cols + col, v[c]);
            float w[V];
            load_weight<T, V>(p.weight, p.weight_f32, col, w);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[c][j] *= w[j];
                if (FP8) gmax[c] = fmaxf(gmax[c], fabsf(v[c][j]));
            }
            if (FP8) amax = fmaxf(amax, gmax[c]);
        }
        if (wide_group) {
            // Maxima do not depend on the order of the atomics (bits of
            // non-negative floats are ordered as integers).
            if (col < p.cols) atomicMax(reinterpret_cast<unsigned int *>(&group_max[col / p.group]), __float_as_uint(gmax[c]));
        } else if (by_group) {
            for (uint32_t m = lanes / 2; m > 0; m >>= 1) gmax[c] = fmaxf(gmax[c], shfl_xor(gmax[c], m));
        }
    }
    row_fold<true>(ss, amax, warp_rows, red);
    if (wide_group) __syncthreads();
    const float rstd = rsqrtf(ss / p.cols + p.eps);
    // |w s| rstd rounds monotonically, so the maximum of |y| is the rounded
    // product of the maximum of |w s|.
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t col = c * step + t * V;
        if (col >= p.cols) continue;
        const int64_t at = (int64_t)row * p.cols + col;
#pragma unroll
        for (int j = 0; j < V; ++j) v[c][j] *= rstd;
        if constexpr (FP8) {
            const uint32_t g = by_group ? col / p.group : 0;
            const float scale = scale_of((wide_group ? group_max[g] : by_group ? gmax[c] : amax) * rstd);
            const float inv = 1.0f / scale;
#pragma unroll
            for (int j = 0; j < V; ++j) v[c][j] *= inv;
            store_fp8<V>(static_cast<uint8_t *>(p.y) + at, v[c]);
            if (col == g * p.group) p.scales[(int64_t)row * p.groups + g] = scale;
        } else {
            store_as<T, V>(static_cast<T *>(p.y) + at, v[c]);
        }
    }
}

// Rows too long for the registers: read twice, the second time from L2.
template <typename T, int V, bool FP8> __global__ void __launch_bounds__(1024) norm_long_kernel(NormParams p) {
    extern __shared__ float group_max[];
    __shared__ float red[2][32];
    const uint32_t row = blockIdx.x, t = threadIdx.x;
    const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
    const T *res = p.residual ? static_cast<const T *>(p.residual) + row * p.residual_stride : nullptr;
    const bool by_group = FP8 && p.groups > 1;
    if (by_group) {
        for (uint32_t g = t; g < p.groups; g += blockDim.x) group_max[g] = 0.0f;
        __syncthreads();
    }
    auto load = [&](uint32_t col, float (&v)[V]) {
        const auto u = *reinterpret_cast<const Pack<T, V> *>(x + col);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = to_f32(u.e[j]);
        if (res) {
            const auto r = *reinterpret_cast<const Pack<T, V> *>(res + col);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] += to_f32(r.e[j]);
        }
    };
    float ss = 0.0f, amax = 0.0f;
    for (uint32_t col = t * V; col < p.cols; col += blockDim.x * V) {
        float v[V], w[V], vmax = 0.0f;
        load(col, v);
        if (res) store_as<T, V>(static_cast<T *>(p.sum) + (int64_t)row * p.cols + col, v);
#pragma unroll
        for (int j = 0; j < V; ++j) ss += v[j] * v[j];
        if constexpr (FP8) {
            load_weight<T, V>(p.weight, p.weight_f32, col, w);
#pragma unroll
            for (int j = 0; j < V; ++j) vmax = fmaxf(vmax, fabsf(v[j] * w[j]));
            amax = fmaxf(amax, vmax);
            if (by_group) atomicMax(reinterpret_cast<unsigned int *>(&group_max[col / p.group]), __float_as_uint(vmax));
        }
    }
    row_fold<true>(ss, amax, false, red);
    if (by_group) __syncthreads();
    const float rstd = rsqrtf(ss / p.cols + p.eps);
    for (uint32_t col = t * V; col < p.cols; col += blockDim.x * V) {
        float v[V], w[V];
        load(col, v);
        load_weight<T, V>(p.weight, p.weight_f32, col, w);
        const int64_t at = (int64_t)row * p.cols + col;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = v[j] * w[j] * rstd;
        if constexpr (FP8) {
            const uint32_t g = by_group ? col / p.group : 0;
            const float scale = scale_of((by_group ? group_max[g] : amax) * rstd);
            const float inv = 1.0f / scale;
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] *= inv;
            store_fp8<V>(static_cast<uint8_t *>(p.y) + at, v);
            if (col == g * p.group) p.scales[(int64_t)row * p.groups + g] = scale;
        } else {
            store_as<T, V>(static_cast<T *>(p.y) + at, v);
        }
    }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned_rows(const Rows &r, size_t es) { return aligned16(r.ptr) && (r.stride * (int64_t)es) % 16 == 0; }

template <typename T, int V, bool FP8> heph_status launch_norm(const NormParams &p, cudaStream_t stream) {
    constexpr int kMost = V == 1 ? 16 : 32 / V;  // values per thread: 16 or 32 registers
    const uint32_t units = p.cols / V;
    const size_t smem = FP8 && p.groups > 1 ? p.groups * sizeof(float) : 0;
    uint32_t c = 1;
    while (c < kMost && (units + c - 1) / c > 256) c *= 2;
    const uint32_t threads = ((units + c - 1) / c + 31) / 32 * 32;
    if (threads > 1024)
        return launch_rows("long row norm", norm_long_kernel<T, V, FP8>, dim3(p.rows), dim3(1024), smem, stream, p);
    // Short rows: one warp each, eight to a block.
    const uint32_t per_block = threads == 32 && !(FP8 && p.groups > 1 && p.group / V > 32) ? 8 : 1;
    const dim3 grid((p.rows + per_block - 1) / per_block), block(threads, per_block);
    auto go = [&](auto kernel) { return launch_rows("row norm", kernel, grid, block, smem, stream, p); };
    switch (c) {
        case 1: return go(norm_kernel<T, V, 1, FP8>);
        case 2: return go(norm_kernel<T, V, 2, FP8>);
        case 4: return go(norm_kernel<T, V, 4, FP8>);
        case 8:
            if constexpr (kMost >= 8) return go(norm_kernel<T, V, 8, FP8>);
            break;
        default:
            if constexpr (kMost >= 16) return go(norm_kernel<T, V, 16, FP8>);
    }
    return fail(HEPH_DISPATCH_FAILED, "no row norm kernel for this width");
}

// ---------------------------------------------------------------- gradient

struct NormGradParams {
    const void *dy, *x, *dsum, *weight;
    void *dx;
    float *partials;
    int64_t dy_stride, x_stride, dsum_stride;
    float eps;
    uint32_t rows, cols;
    bool weight_f32;
};

// Block b takes rows b, b + gridDim.x, ...; its share of dw stays in
// registers (each thread keeps its columns) and goes out once.
template <typename T, int V, int C>
__global__ void __launch_bounds__(512) norm_grad_kernel(NormGradParams p) {
    __shared__ float red[2][2][32];
    const uint32_t t = threadIdx.x, step = blockDim.x * V;
    float dw[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) dw[c][j] = 0.0f;
    uint32_t turn = 0;
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const T *dy = static_cast<const T *>(p.dy) + row * p.dy_stride;
        const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
        Pack<T, V> ug[C], ux[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint32_t col = c * step + t * V;
            if (col < p.cols) {
                ug[c] = *reinterpret_cast<const Pack<T, V> *>(dy + col);
                ux[c] = *reinterpret_cast<const Pack<T, V> *>(x + col);
            }
        }
        float ss = 0.0f, gs = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint32_t col = c * step + t * V;
            if (col < p.cols) {
                float w[V];
                load_weight<T, V>(p.weight, p.weight_f32, col, w);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float s = to_f32(ux[c].e[j]);
                    ss += s * s;
                    gs += to_f32(ug[c].e[j]) * w[j] * s;
                }
            }
        }
        row_fold<false>(ss, gs, false, red[turn]);  // two buffers: one barrier per row is enough
        const float rstd = rsqrtf(ss / p.cols + p.eps);
        const float back = rstd * rstd * (gs / p.cols);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint32_t col = c * step + t * V;
            if (col < p.cols) {
                float w[V], dx[V];
                load_weight<T, V>(p.weight, p.weight_f32, col, w);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float s = to_f32(ux[c].e[j]), g = to_f32(ug[c].e[j]);
                    dw[c][j] += g * s * rstd;
                    dx[j] = rstd * (g * w[j] - s * back);
                }
                if (p.dsum) {
                    const auto u = *reinterpret_cast<const Pack<T, V> *>(static_cast<const T *>(p.dsum) +
                                                                         row * p.dsum_stride + col);
#pragma unroll
                    for (int j = 0; j < V; ++j) dx[j] += to_f32(u.e[j]);
                }
                store_as<T, V>(static_cast<T *>(p.dx) + (int64_t)row * p.cols + col, dx);
            }
        }
    }
    if (!p.partials) return;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t col = c * step + t * V;
        if (col < p.cols) {
#pragma unroll
            for (int j = 0; j < V; ++j) p.partials[(int64_t)blockIdx.x * p.cols + col + j] = dw[c][j];
        }
    }
}

// Rows too long for the registers: read twice; the block's share of dw is
// gathered in its own row of `partials`, each thread its own columns.
template <typename T> __global__ void __launch_bounds__(1024) norm_grad_long_kernel(NormGradParams p) {
    __shared__ float red[2][2][32];
    uint32_t turn = 0;
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const T *dy = static_cast<const T *>(p.dy) + row * p.dy_stride;
        const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
        float ss = 0.0f, gs = 0.0f;
        for (uint32_t col = threadIdx.x; col < p.cols; col += blockDim.x) {
            float w[1];
            load_weight<T, 1>(p.weight, p.weight_f32, col, w);
            const float s = to_f32(x[col]);
            ss += s * s;
            gs += to_f32(dy[col]) * w[0] * s;
        }
        row_fold<false>(ss, gs, false, red[turn]);
        const float rstd = rsqrtf(ss / p.cols + p.eps);
        const float back = rstd * rstd * (gs / p.cols);
        for (uint32_t col = threadIdx.x; col < p.cols; col += blockDim.x) {
            float w[1];
            load_weight<T, 1>(p.weight, p.weight_f32, col, w);
            const float s = to_f32(x[col]), g = to_f32(dy[col]);
            float dx = rstd * (g * w[0] - s * back);
            if (p.dsum) dx += to_f32(static_cast<const T *>(p.dsum)[row * p.dsum_stride + col]);
            static_cast<T *>(p.dx)[(int64_t)row * p.cols + col] = from_f32<T>(dx);
            if (p.partials) {
                float *mine = p.partials + (int64_t)blockIdx.x * p.cols + col;
                *mine = (row == blockIdx.x ? 0.0f : *mine) + g * s * rstd;
            }
        }
    }
}

// dw[col] = sum of the partial rows, in the same order on every call: eight
// warps of a block each fold every eighth row of 32 columns.
template <typename W> __global__ void __launch_bounds__(256) norm_dweight_kernel(const float *partials, uint32_t parts,
                                                                                 uint32_t cols, W *dweight) {
    __shared__ float part[8][33];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
    float sum = 0.0f;
    if (col < cols) {
#pragma unroll 8
        for (uint32_t r = warp; r < parts; r += 8) sum += partials[(int64_t)r * cols + col];
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && col < cols) {
#pragma unroll
        for (int w = 1; w < 8; ++w) sum += part[w][lane];
        dweight[col] = from_f32<W>(sum);
    }
}

template <typename T, int V> heph_status launch_norm_grad(const NormGradParams &p, uint32_t blocks, cudaStream_t stream) {
    constexpr int kMost = 32 / V;
    const uint32_t units = p.cols / V;
    uint32_t c = 1;
    while (c < kMost && (units + c - 1) / c > 256) c *= 2;
    const uint32_t threads = ((units + c - 1) / c + 31) / 32 * 32;
    if (threads > 512)
        return launch_rows("long row norm gradient", norm_grad_long_kernel<T>, dim3(blocks), dim3(1024), 0, stream, p);
    auto go = [&](auto kernel) { return launch_rows("row norm gradient", kernel, dim3(blocks), dim3(threads), 0, stream, p); };
    switch (c) {
        case 1: return go(norm_grad_kernel<T, V, 1>);
        case 2: return go(norm_grad_kernel<T, V, 2>);
        case 4: return go(norm_grad_kernel<T, V, 4>);
        case 8:
            if constexpr (kMost >= 8) return go(norm_grad_kernel<T, V, 8>);
            break;
        case 16:
            if constexpr (kMost >= 16) return go(norm_grad_kernel<T, V, 16>);
            break;
        default:
            if constexpr (kMost >= 32) return go(norm_grad_kernel<T, V, 32>);
    }
    return fail(HEPH_DISPATCH_FAILED, "no row norm gradient kernel for this width");
}

}  // namespace

heph_status launch_rms_norm(const NormArgs &a, cudaStream_t stream) {
    const bool fp8 = a.scales != nullptr;
    const uint32_t group = a.group && a.group < a.cols ? a.group : a.cols;
    const NormParams p{a.x.ptr, a.residual.ptr, a.weight, a.y, a.sum, a.scales, a.x.stride, a.residual.stride, a.eps,
                       a.rows, a.cols, group, (a.cols + group - 1) / group, a.weight_f32};
    return dispatch_row_dtype(a.dtype, [&]<typename T>() {
        constexpr int V = 16 / sizeof(T);
        // 16-byte accesses need every row of every operand to start on one.
        const bool wide = a.cols % V == 0 && aligned_rows(a.x, sizeof(T)) && aligned_rows(a.residual, sizeof(T)) &&
                          aligned16(a.weight) && aligned16(a.y) && aligned16(a.sum);
        if (fp8) return wide ? launch_norm<T, V, true>(p, stream) : launch_norm<T, 1, true>(p, stream);
        return wide ? launch_norm<T, V, false>(p, stream) : launch_norm<T, 1, false>(p, stream);
    });
}

uint32_t norm_grad_partials(uint32_t rows, int sm_count) { return std::min<uint32_t>(rows, 2 * sm_count); }

heph_status launch_rms_norm_backward(const NormGradArgs &a, int sm_count, cudaStream_t stream) {
    const uint32_t blocks = norm_grad_partials(a.rows, sm_count);
    const NormGradParams p{a.dy.ptr, a.x.ptr, a.dsum.ptr, a.weight, a.dx, a.dweight ? a.partials : nullptr, a.dy.stride,
                           a.x.stride, a.dsum.stride, a.eps, a.rows, a.cols, a.weight_f32};
    return dispatch_row_dtype(a.dtype, [&]<typename T>() {
        constexpr int V = 16 / sizeof(T);
        if (a.rows) {
            const bool wide = a.cols % V == 0 && aligned_rows(a.dy, sizeof(T)) && aligned_rows(a.x, sizeof(T)) &&
                              aligned_rows(a.dsum, sizeof(T)) && aligned16(a.weight) && aligned16(a.dx);
            const heph_status st = wide ? launch_norm_grad<T, V>(p, blocks, stream) : launch_norm_grad<T, 1>(p, blocks, stream);
            if (st != HEPH_OK) return st;
        }
        if (!a.dweight) return HEPH_OK;
        const dim3 grid((a.cols + 31) / 32);
        auto fold = [&](auto *dw) {
            return launch_rows("norm weight gradient", norm_dweight_kernel<std::remove_pointer_t<decltype(dw)>>, grid,
                               dim3(256), 0, stream, a.partials, blocks, a.cols, dw);
        };
        return a.weight_f32 ? fold(static_cast<float *>(a.dweight)) : fold(static_cast<T *>(a.dweight));
    });
}

}  // namespace heph
