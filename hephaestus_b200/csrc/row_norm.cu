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
    float eps, per_col;  // per_col = 1 / cols
    uint32_t rows, cols;
    uint32_t group_shift, groups;  // 2^shift columns per scale, scales per row
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

// 16 bytes into shared memory past the registers; groups of copies complete
// for the thread that asked for them, in order.
__device__ __forceinline__ void copy16_async(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// How the scales are made.
enum Scales : int {
    kNoScales,     // output in the rows' type
    kRowScale,     // one for the row
    kLaneScales,   // groups of a power of two of lanes, up to a warp
    kSharedScales  // any group, its maximum in shared memory
};

// Sum of a and maximum (MAX) or sum of b over the block, or over the warp
// when rows are warps; every thread gets both.  One barrier.
template <bool TWO, bool MAX>
__device__ __forceinline__ void row_fold(float &a, float &b, bool warp_rows, float2 *red) {
    a = warp_sum(a);
    if (TWO) b = MAX ? warp_max(b) : warp_sum(b);
    if (warp_rows || blockDim.x == 32) return;
    const uint32_t lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) red[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    // Up to 8 warps are folded by every 8 lanes.
    const uint32_t from = warps <= 8 ? lane & 7 : lane;
    const float2 o = from < warps ? red[from] : make_float2(0.0f, 0.0f);
    a = o.x;
    b = o.y;
    for (uint32_t m = warps <= 8 ? 4 : 16; m > 0; m >>= 1) {
        a += shfl_xor(a, m);
        if (TWO) b = MAX ? fmaxf(b, shfl_xor(b, m)) : b + shfl_xor(b, m);
    }
}

__device__ __forceinline__ void shared_max(float *at, float v) {
    // Maxima do not depend on the order of the atomics (bits of non-negative
    // floats are ordered as integers).
    atomicMax(reinterpret_cast<unsigned int *>(at), __float_as_uint(v));
}
__device__ __forceinline__ float scale_of(float amax) { return fmaxf(amax, kFp8Floor) * (1.0f / kFp8Max); }

// A row (or, blockDim.y > 1, a row per warp) whose C x V values per thread
// stay in registers between the one read and the one write.
//
// SHIFTED: rows of odd widths.  Row r of every operand starts the same number
// of elements past a 16-byte boundary; accesses are whole vectors from
// boundary to boundary, but for the row's two ends (and the weights, whose
// boundaries are elsewhere: element by element, from L1).
template <typename T, int V, int C, Scales S, bool RES, bool SHIFTED>
__global__ void __launch_bounds__(C * V >= 32 ? 512 : 1024) norm_kernel(const __grid_constant__ NormParams p) {
    extern __shared__ float group_max[];  // kSharedScales: of each group
    __shared__ float2 red[32];
    const bool warp_rows = blockDim.y > 1;
    const uint32_t row = blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= p.rows) return;  // whole warps, which no block barrier waits for
    const uint32_t t = threadIdx.x, step = blockDim.x * V;
    const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
    const T *res = RES ? static_cast<const T *>(p.residual) + row * p.residual_stride : nullptr;
    T *sum = RES ? static_cast<T *>(p.sum) + (int64_t)row * p.cols : nullptr;
    // Columns of this thread's chunk c: first, first + 1, ...; a SHIFTED row's
    // first chunk starts before column 0 (and the unsigned number wraps).
    const uint32_t lead = SHIFTED ? (uint32_t)(reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T) : 0;
    auto first = [&](int c) { return c * step + t * V - lead; };
    auto whole = [&](uint32_t col) { return SHIFTED ? col < p.cols && col + V <= p.cols : col < p.cols; };
    auto some = [&](uint32_t col) { return SHIFTED && col + V - 1 < p.cols + V - 1; };  // part of it, or all
    if (S == kSharedScales) {
        for (uint32_t g = t; g < p.groups; g += blockDim.x) group_max[g] = 0.0f;
        __syncthreads();
    }

    Pack<T, V> ux[C], ur[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t col = first(c);
        if (whole(col)) {
            ux[c] = *reinterpret_cast<const Pack<T, V> *>(x + col);
            if (RES) ur[c] = *reinterpret_cast<const Pack<T, V> *>(res + col);
        } else if (some(col)) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                ux[c].e[j] = col + j < p.cols ? x[col + j] : from_f32<T>(0.0f);
                if (RES) ur[c].e[j] = col + j < p.cols ? res[col + j] : from_f32<T>(0.0f);
            }
        }
    }
    float v[C][V], ss = 0.0f, amax = 0.0f, gmax[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t col = first(c);
        gmax[c] = 0.0f;
        if (whole(col) || some(col)) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[c][j] = to_f32(ux[c].e[j]);
                if (RES) v[c][j] += to_f32(ur[c].e[j]);
                ss += v[c][j] * v[c][j];
            }
            if (RES) {
                if (whole(col)) {
                    store_as<T, V>(sum + col, v[c]);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (col + j < p.cols) sum[col + j] = from_f32<T>(v[c][j]);
                }
            }
            if (SHIFTED) {
                if (p.weight) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        float w[1] = {0.0f};
                        if (col + j < p.cols) load_weight<T, 1>(p.weight, p.weight_f32, col + j, w);
                        v[c][j] *= w[0];
                    }
                }
            } else {
                float w[V];
                load_weight<T, V>(p.weight, p.weight_f32, col, w);
#pragma unroll
                for (int j = 0; j < V; ++j) v[c][j] *= w[j];
            }
            if (S == kRowScale || S == kLaneScales || (S == kSharedScales && !SHIFTED)) {
#pragma unroll
                for (int j = 0; j < V; ++j) gmax[c] = fmaxf(gmax[c], fabsf(v[c][j]));
                amax = fmaxf(amax, gmax[c]);
                if (S == kSharedScales) shared_max(&group_max[col >> p.group_shift], gmax[c]);
            } else if (S == kSharedScales) {
                // Two groups at most: of the first and of the last column.
                const uint32_t g = (col < p.cols ? col : 0) >> p.group_shift;
                float a = 0.0f, b = 0.0f;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const bool next = col + j < p.cols && (col + j) >> p.group_shift != g;
                    a = fmaxf(a, next ? 0.0f : fabsf(v[c][j]));
                    b = fmaxf(b, next ? fabsf(v[c][j]) : 0.0f);
                }
                shared_max(&group_max[g], a);
                if (b > 0.0f) shared_max(&group_max[g + 1], b);
            }
        }
        if (S == kLaneScales) {
            for (uint32_t m = (1u << p.group_shift) / V / 2; m > 0; m >>= 1) gmax[c] = fmaxf(gmax[c], shfl_xor(gmax[c], m));
        }
    }
    row_fold<S == kRowScale, true>(ss, amax, warp_rows, red);
    if (S == kSharedScales) __syncthreads();
    const float rstd = rsqrtf(ss * p.per_col + p.eps);
    // |w s| rstd rounds monotonically, so the maximum of |y| is the rounded
    // product of the maximum of |w s|.
    float scale, factor = rstd;
    if (S == kRowScale) {
        scale = scale_of(amax * rstd);
        factor = rstd * __fdividef(1.0f, scale);
        if (t == 0) p.scales[row] = scale;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t col = first(c);
        if (!whole(col) && !some(col)) continue;
        const int64_t at = (int64_t)row * p.cols + (int32_t)col;
        if (S == kLaneScales || (S == kSharedScales && !SHIFTED)) {
            const uint32_t g = col >> p.group_shift;
            scale = scale_of((S == kLaneScales ? gmax[c] : group_max[g]) * rstd);
            factor = rstd * __fdividef(1.0f, scale);
            if (col == g << p.group_shift) p.scales[(int64_t)row * p.groups + g] = scale;
        }
        if (S == kSharedScales && SHIFTED) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (col + j >= p.cols) continue;
                const uint32_t g = (col + j) >> p.group_shift;
                scale = scale_of(group_max[g] * rstd);
                v[c][j] *= rstd * __fdividef(1.0f, scale);
                if (col + j == g << p.group_shift) p.scales[(int64_t)row * p.groups + g] = scale;
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[c][j] *= factor;
        }
        if constexpr (S != kNoScales) {
            if (!SHIFTED) {
                store_fp8<V>(static_cast<uint8_t *>(p.y) + at, v[c]);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float one[1] = {v[c][j]};
                    if (col + j < p.cols) store_fp8<1>(static_cast<uint8_t *>(p.y) + at + j, one);
                }
            }
        } else if (whole(col)) {
            store_as<T, V>(static_cast<T *>(p.y) + at, v[c]);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (col + j < p.cols) static_cast<T *>(p.y)[at + j] = from_f32<T>(v[c][j]);
        }
    }
}

// Rows too long for the registers, or of operands with no common boundaries:
// read twice, the second time from L2.
template <typename T, int V, bool FP8> __global__ void __launch_bounds__(1024) norm_long_kernel(const __grid_constant__ NormParams p) {
    extern __shared__ float group_max[];
    __shared__ float2 red[32];
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
#pragma unroll 2
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
            if (by_group) shared_max(&group_max[col >> p.group_shift], vmax);
        }
    }
    row_fold<FP8, true>(ss, amax, false, red);
    if (by_group) __syncthreads();
    const float rstd = rsqrtf(ss * p.per_col + p.eps);
#pragma unroll 2
    for (uint32_t col = t * V; col < p.cols; col += blockDim.x * V) {
        float v[V], w[V];
        load(col, v);
        load_weight<T, V>(p.weight, p.weight_f32, col, w);
        const int64_t at = (int64_t)row * p.cols + col;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] *= w[j];
        if constexpr (FP8) {
            const uint32_t g = by_group ? col >> p.group_shift : 0;
            const float scale = scale_of((by_group ? group_max[g] : amax) * rstd);
            const float factor = rstd * __fdividef(1.0f, scale);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] *= factor;
            store_fp8<V>(static_cast<uint8_t *>(p.y) + at, v);
            if (by_group ? col == g << p.group_shift : col == 0) p.scales[(int64_t)row * p.groups + g] = scale;
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] *= rstd;
            store_as<T, V>(static_cast<T *>(p.y) + at, v);
        }
    }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned_rows(const Rows &r, size_t es) { return aligned16(r.ptr) && (r.stride * (int64_t)es) % 16 == 0; }

// SHIFTED (see norm_kernel) or not: rows of whole vectors.
template <typename T, bool FP8, bool SHIFTED> heph_status launch_norm(const NormParams &p, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    constexpr int kMost = 32 / V;  // chunks of a thread: 32 registers
    const uint32_t units = SHIFTED ? (p.cols + 2 * V - 2) / V : p.cols / V;
    const size_t smem = FP8 && p.groups > 1 ? p.groups * sizeof(float) : 0;
    // Rows of up to 256 threads where the chunks reach, as rows of few warps
    // wait less for one another.
    uint32_t c = 1;
    while (c < kMost && (units + c - 1) / c > 256) c *= 2;
    const uint32_t threads = ((units + c - 1) / c + 31) / 32 * 32;
    if (threads > (c * V >= 32 ? 512 : 1024)) {
        if constexpr (!SHIFTED) return launch_rows("long row norm", norm_long_kernel<T, V, FP8>, dim3(p.rows), dim3(1024), smem, stream, p);
        return launch_rows("long row norm", norm_long_kernel<T, 1, FP8>, dim3(p.rows), dim3(1024), smem, stream, p);
    }
    const bool in_lanes = !SHIFTED && p.groups > 1 && (1u << p.group_shift) / V <= 32;
    // Short rows: one warp each, eight to a block (not where they share group_max).
    const uint32_t per_block = threads == 32 && (!FP8 || p.groups == 1 || in_lanes) ? 8 : 1;
    const dim3 grid((p.rows + per_block - 1) / per_block), block(threads, per_block);
    auto scaled = [&]<int C, Scales S>() {
        auto kernel = p.residual ? norm_kernel<T, V, C, S, true, SHIFTED> : norm_kernel<T, V, C, S, false, SHIFTED>;
        return launch_rows("row norm", kernel, grid, block, smem, stream, p);
    };
    auto go = [&]<int C>() {
        if constexpr (!FP8) {
            return scaled.template operator()<C, kNoScales>();
        } else {
            if (p.groups == 1) return scaled.template operator()<C, kRowScale>();
            if constexpr (!SHIFTED) {
                if (in_lanes) return scaled.template operator()<C, kLaneScales>();
            }
            return scaled.template operator()<C, kSharedScales>();
        }
    };
    switch (c) {
        case 1: return go.template operator()<1>();
        case 2: return go.template operator()<2>();
        case 4: return go.template operator()<4>();
        default:
            if constexpr (kMost >= 8) return go.template operator()<8>();
    }
    return fail(HEPH_DISPATCH_FAILED, "no row norm kernel for this width");
}

// ---------------------------------------------------------------- gradient

struct NormGradParams {
    const void *dy, *x, *dsum, *weight;
    void *dx;
    float *partials;
    int64_t dy_stride, x_stride, dsum_stride;
    float eps, per_col;
    uint32_t rows, cols;
    bool weight_f32;
};

// Block b takes rows b, b + gridDim.x, ...; its share of dw stays in registers
// (each thread keeps its columns) and goes out once.
//
// With whole vectors (V > 1) the rows pass through shared memory, kStages - 1
// of them on their way while one is worked on: the registers hold dw and one
// row, and could not hold another.  Each thread copies what it reads itself,
// so a copy needs no barrier but the thread's own wait.
constexpr int kMaxGradSmem = 2 * 3 * 16 * 4 * 512;
template <int C> constexpr int kGradStages = C >= 4 ? 2 : 4;

template <typename T, int V, int C>
__global__ void __launch_bounds__(512) norm_grad_kernel(const __grid_constant__ NormGradParams p) {
    constexpr int kStages = kGradStages<C>;
    using Vector = Pack<T, V>;
    extern __shared__ __align__(16) unsigned char staged[];  // [kStages][3][C][threads] vectors
    __shared__ float2 red[2][16];
    const uint32_t t = threadIdx.x, step = blockDim.x * V;
    const T *dy = static_cast<const T *>(p.dy), *x = static_cast<const T *>(p.x), *dsum = static_cast<const T *>(p.dsum);
    auto slot = [&](uint32_t stage, int operand, int c) {
        return reinterpret_cast<Vector *>(staged) + ((stage * 3 + operand) * C + c) * blockDim.x + t;
    };
    auto request = [&](uint32_t row, uint32_t stage) {
        if constexpr (V > 1) {
            if (row < p.rows) {
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const uint32_t col = c * step + t * V;
                    if (col >= p.cols) continue;
                    copy16_async(slot(stage, 0, c), dy + row * p.dy_stride + col);
                    copy16_async(slot(stage, 1, c), x + row * p.x_stride + col);
                    if (dsum) copy16_async(slot(stage, 2, c), dsum + row * p.dsum_stride + col);
                }
            }
            copies_commit();  // a group for every row, empty ones too
        }
    };
    float dw[C][V];
    Vector uw[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t col = c * step + t * V;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            dw[c][j] = 0.0f;
            uw[c].e[j] = from_f32<T>(1.0f);
        }
        if (p.weight && !p.weight_f32 && col < p.cols)
            uw[c] = *reinterpret_cast<const Vector *>(static_cast<const T *>(p.weight) + col);
    }
    // f32 weights beside 16-bit rows do not fit in uw: read again for each row, from L1.
    auto weight = [&](int c, uint32_t col, float (&w)[V]) {
        if (p.weight_f32) {
            load_weight<T, V>(p.weight, true, col, w);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = to_f32(uw[c].e[j]);
        }
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) request(blockIdx.x + i * gridDim.x, i);
    uint32_t turn = 0, stage = 0;
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        Vector ug[C], ux[C];
        if constexpr (V > 1) {
            copies_wait<kStages - 2>();
            // Into the slot that was read a row ago.
            request(row + (kStages - 1) * gridDim.x, stage == 0 ? kStages - 1 : stage - 1);
        }
        float ss = 0.0f, gs = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint32_t col = c * step + t * V;
            if (col < p.cols) {
                if constexpr (V > 1) {
                    ug[c] = *slot(stage, 0, c);
                    ux[c] = *slot(stage, 1, c);
                } else {
                    ug[c].e[0] = dy[row * p.dy_stride + col];
                    ux[c].e[0] = x[row * p.x_stride + col];
                }
                float w[V];
                weight(c, col, w);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float s = to_f32(ux[c].e[j]);
                    ss += s * s;
                    gs += to_f32(ug[c].e[j]) * w[j] * s;
                }
            }
        }
        row_fold<true, false>(ss, gs, false, red[turn]);  // two buffers: one barrier per row is enough
        const float rstd = rsqrtf(ss * p.per_col + p.eps);
        const float back = rstd * rstd * rstd * (gs * p.per_col);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint32_t col = c * step + t * V;
            if (col < p.cols) {
                float w[V], dx[V] = {};
                if (dsum) {
                    Vector u;
                    if constexpr (V > 1) u = *slot(stage, 2, c);
                    else u.e[0] = dsum[row * p.dsum_stride + col];
#pragma unroll
                    for (int j = 0; j < V; ++j) dx[j] = to_f32(u.e[j]);
                }
                weight(c, col, w);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float s = to_f32(ux[c].e[j]), g = to_f32(ug[c].e[j]) * rstd;
                    dw[c][j] += g * s;
                    dx[j] += g * w[j] - s * back;
                }
                store_as<T, V>(static_cast<T *>(p.dx) + (int64_t)row * p.cols + col, dx);
            }
        }
        stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    if (!p.partials) return;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t col = c * step + t * V;
        if (col < p.cols) store_as<float, V>(p.partials + (int64_t)blockIdx.x * p.cols + col, dw[c]);
    }
}

// Rows too long for the registers: read twice; the block's share of dw is
// gathered in its own row of `partials`, each thread its own columns.
template <typename T, int V> __global__ void __launch_bounds__(1024) norm_grad_long_kernel(const __grid_constant__ NormGradParams p) {
    __shared__ float2 red[2][32];
    uint32_t turn = 0;
    auto load = [](const void *src, int64_t at, float (&v)[V]) {
        const auto u = *reinterpret_cast<const Pack<T, V> *>(static_cast<const T *>(src) + at);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = to_f32(u.e[j]);
    };
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        float ss = 0.0f, gs = 0.0f;
        for (uint32_t col = threadIdx.x * V; col < p.cols; col += blockDim.x * V) {
            float w[V], s[V], g[V];
            load_weight<T, V>(p.weight, p.weight_f32, col, w);
            load(p.x, row * p.x_stride + col, s);
            load(p.dy, row * p.dy_stride + col, g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                ss += s[j] * s[j];
                gs += g[j] * w[j] * s[j];
            }
        }
        row_fold<true, false>(ss, gs, false, red[turn]);
        const float rstd = rsqrtf(ss * p.per_col + p.eps);
        const float back = rstd * rstd * rstd * (gs * p.per_col);
        for (uint32_t col = threadIdx.x * V; col < p.cols; col += blockDim.x * V) {
            float w[V], s[V], g[V], dx[V] = {};
            load_weight<T, V>(p.weight, p.weight_f32, col, w);
            load(p.x, row * p.x_stride + col, s);
            load(p.dy, row * p.dy_stride + col, g);
            if (p.dsum) load(p.dsum, row * p.dsum_stride + col, dx);
            float *mine = p.partials ? p.partials + (int64_t)blockIdx.x * p.cols + col : nullptr;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                dx[j] += g[j] * rstd * w[j] - s[j] * back;
                if (mine) mine[j] = (row == blockIdx.x ? 0.0f : mine[j]) + g[j] * rstd * s[j];
            }
            store_as<T, V>(static_cast<T *>(p.dx) + (int64_t)row * p.cols + col, dx);
        }
    }
}

// dw[col] = sum of the partial rows, in the same order on every call: each of
// 32 warps folds every 32nd row of 32 columns.
template <typename W> __global__ void __launch_bounds__(1024) norm_dweight_kernel(const float *partials, uint32_t parts,
                                                                                  uint32_t cols, W *dweight) {
    __shared__ float part[32][33];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
    float sum = 0.0f;
    if (col < cols) {
#pragma unroll 8
        for (uint32_t r = warp; r < parts; r += 32) sum += partials[(int64_t)r * cols + col];
    }
    part[warp][lane] = sum;
    __syncthreads();
    sum = warp_sum(part[lane][warp]);  // of column `warp`
    const uint32_t mine = blockIdx.x * 32 + warp;
    if (lane == 0 && mine < cols) dweight[mine] = from_f32<W>(sum);
}

template <typename T, int V>
heph_status launch_norm_grad(const NormGradParams &p, uint32_t partials, int sm_count, uint32_t *out_blocks, cudaStream_t stream) {
    constexpr int kMost = 16 / V;  // chunks of a thread: 16 registers for each of five vectors
    const uint32_t units = p.cols / V;
    uint32_t c = 1;
    while (c < kMost && (units + c - 1) / c > 256) c *= 2;
    const uint32_t threads = ((units + c - 1) / c + 31) / 32 * 32;
    // As many blocks as run at once: two an SM of up to 256 threads, else one.
    const uint32_t blocks = *out_blocks = threads <= 256 ? partials : std::min<uint32_t>(partials, sm_count);
    if (threads > 512)
        return launch_rows("long row norm gradient", norm_grad_long_kernel<T, V>, dim3(blocks), dim3(1024), 0, stream, p);
    auto go = [&]<int C>() -> heph_status {
        const size_t smem = V > 1 ? kGradStages<C> * 3 * 16 * C * threads : 0;
        if (smem)
            HEPH_CUDA_TRY(cudaFuncSetAttribute(norm_grad_kernel<T, V, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxGradSmem),
                          HEPH_DISPATCH_FAILED, "row norm gradient shared memory");
        return launch_rows("row norm gradient", norm_grad_kernel<T, V, C>, dim3(blocks), dim3(threads), smem, stream, p);
    };
    switch (c) {
        case 1: return go.template operator()<1>();
        case 2: return go.template operator()<2>();
        case 4:
            if constexpr (kMost >= 4) return go.template operator()<4>();
            break;
        case 8:
            if constexpr (kMost >= 8) return go.template operator()<8>();
            break;
        default:
            if constexpr (kMost >= 16) return go.template operator()<16>();
    }
    return fail(HEPH_DISPATCH_FAILED, "no row norm gradient kernel for this width");
}

}  // namespace

heph_status launch_rms_norm(const NormArgs &a, cudaStream_t stream) {
    const bool fp8 = a.scales != nullptr;
    const bool grouped = fp8 && a.group && a.group < a.cols;
    const uint32_t shift = grouped ? __builtin_ctz(a.group) : 31;
    const NormParams p{a.x.ptr, a.residual.ptr, a.weight, a.y, a.sum, a.scales, a.x.stride, a.residual.stride, a.eps,
                       1.0f / a.cols, a.rows, a.cols, shift, grouped ? (a.cols + a.group - 1) / a.group : 1, a.weight_f32};
    return dispatch_row_dtype(a.dtype, [&]<typename T>() {
        constexpr int V = 16 / sizeof(T);
        // Whole vectors need every row of every operand to start on 16 bytes.
        const bool wide = a.cols % V == 0 && aligned_rows(a.x, sizeof(T)) && aligned_rows(a.residual, sizeof(T)) &&
                          aligned16(a.weight) && aligned16(a.y) && aligned16(a.sum);
        if (wide) return fp8 ? launch_norm<T, true, false>(p, stream) : launch_norm<T, false, false>(p, stream);
        // Shifted ones, the same distance past a boundary in every operand of
        // the rows' type (e4m3 is written by the byte).
        auto like = [&](const void *ptr, int64_t stride) {
            const auto apart = reinterpret_cast<intptr_t>(ptr) - reinterpret_cast<intptr_t>(a.x.ptr);
            return !ptr || (apart % 16 == 0 && (stride - a.x.stride) % V == 0);
        };
        const bool shifted = like(a.residual.ptr, a.residual.stride) && like(a.sum, a.cols) && (fp8 || like(a.y, a.cols));
        if (shifted) return fp8 ? launch_norm<T, true, true>(p, stream) : launch_norm<T, false, true>(p, stream);
        const size_t smem = p.groups > 1 ? p.groups * sizeof(float) : 0;
        auto kernel = fp8 ? norm_long_kernel<T, 1, true> : norm_long_kernel<T, 1, false>;
        return launch_rows("row norm", kernel, dim3(p.rows), dim3(std::min(1024u, (p.cols + 127) / 128 * 32)), smem, stream, p);
    });
}

uint32_t norm_grad_partials(uint32_t rows, int sm_count) { return std::min<uint32_t>(rows, 2 * sm_count); }

heph_status launch_rms_norm_backward(const NormGradArgs &a, int sm_count, cudaStream_t stream) {
    const uint32_t partials = norm_grad_partials(a.rows, sm_count);
    uint32_t blocks = 0;  // of these used
    const NormGradParams p{a.dy.ptr, a.x.ptr, a.dsum.ptr, a.weight, a.dx, a.dweight ? a.partials : nullptr, a.dy.stride,
                           a.x.stride, a.dsum.stride, a.eps, 1.0f / a.cols, a.rows, a.cols, a.weight_f32};
    return dispatch_row_dtype(a.dtype, [&]<typename T>() {
        constexpr int V = 16 / sizeof(T);
        if (a.rows) {
            const bool wide = a.cols % V == 0 && aligned_rows(a.dy, sizeof(T)) && aligned_rows(a.x, sizeof(T)) &&
                              aligned_rows(a.dsum, sizeof(T)) && aligned16(a.weight) && aligned16(a.dx);
            const heph_status st = wide ? launch_norm_grad<T, V>(p, partials, sm_count, &blocks, stream)
                                        : launch_norm_grad<T, 1>(p, partials, sm_count, &blocks, stream);
            if (st != HEPH_OK) return st;
        }
        if (!a.dweight) return HEPH_OK;
        const dim3 grid((a.cols + 31) / 32);
        auto fold = [&](auto *dw) {
            return launch_rows("norm weight gradient", norm_dweight_kernel<std::remove_pointer_t<decltype(dw)>>, grid,
                               dim3(1024), 0, stream, a.partials, blocks, a.cols, dw);
        };
        return a.weight_f32 ? fold(static_cast<float *>(a.dweight)) : fold(static_cast<T *>(a.dweight));
    });
}

}  // namespace heph
