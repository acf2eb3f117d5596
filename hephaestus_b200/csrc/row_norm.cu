// row_norm.cu — root-mean-square norm of rows, with the residual's addition
// and 8-bit output, and its gradient.
//
//   s = x + residual,  rstd = 1 / sqrt(mean(s^2) + eps),  y = w s rstd
//   e4m3 output: scale = max(max|y|, 2^-100) / 448 over a row or a group of
//   columns, q = y / scale.
//   gradient:    dx = rstd (w dy - xhat mean(w dy xhat)) + dsum, xhat = s rstd,
//                dw = sum over rows of dy xhat
//
// No power of rstd is formed: its cube leaves 32 bits where the result does not
// (rows of rms above 4e12 or below 2e-13).
//
// All in 32 bits from the unrounded sum s; each output is rounded once.
#include <cuda_fp8.h>

#include <algorithm>
#include <initializer_list>

#include "row_ops.h"
#include "row_utils.cuh"

namespace heph {

namespace {

constexpr float kFp8Max = 448.0f;       // largest finite e4m3 value
// Smallest maximum a scale is made for: keeps 1 / scale finite.  Its product
// with rstd need not be, so values take rstd first and 1 / scale then.
constexpr float kFp8Floor = 0x1p-100f;

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

// Accesses of 16 bytes at most: what operands and the workspace are aligned to.
template <typename T, int V> __device__ __forceinline__ void store_as(T *dst, const float (&v)[V]) {
    constexpr int N = V * sizeof(T) <= 16 ? V : 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < V / N; ++i) {
        Pack<T, N> u;
#pragma unroll
        for (int j = 0; j < N; ++j) u.e[j] = from_f32<T>(v[i * N + j]);
        *reinterpret_cast<Pack<T, N> *>(dst + i * N) = u;
    }
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

// Columns of a thread's chunks of V, `step` apart.  SHIFTED: rows of odd widths.
// Row r of every operand starts the same number of elements past a 16-byte
// boundary, `lead`; chunks go from boundary to boundary, and the row's two
// ends, which are parts of chunks, are taken element by element.
template <int V, int C, bool SHIFTED> struct Chunks {
    uint32_t cols, step, origin;
    uint32_t wholes = 0, somes = 0;  // SHIFTED chunks that lie in the row, and of which some column does, a bit each
    __device__ Chunks(uint32_t cols_, const void *row, size_t size)
        : cols(cols_), step(blockDim.x * V),
          origin(threadIdx.x * V - (SHIFTED ? (uint32_t)((reinterpret_cast<uintptr_t>(row) & 15u) / size) : 0)) {
        if (!SHIFTED) return;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint32_t col = first(c);
            wholes |= (col < cols && col + V <= cols ? 1u : 0u) << c;
            somes |= (col + V - 1 < cols + V - 1 ? 1u : 0u) << c;
        }
    }
    // Chunk c's first column; a SHIFTED row's first chunk starts before column
    // 0, and the number wraps.
    __device__ __forceinline__ uint32_t first(int c) const { return c * step + origin; }
    __device__ __forceinline__ bool whole(int c) const { return SHIFTED ? wholes >> c & 1u : first(c) < cols; }
    __device__ __forceinline__ bool some(int c) const { return SHIFTED ? somes >> c & 1u : first(c) < cols; }
    __device__ __forceinline__ bool has(uint32_t col, int j) const { return !SHIFTED || col + j < cols; }

    template <typename T> __device__ __forceinline__ Pack<T, V> load(const T *row, int c) const {
        const uint32_t col = first(c);
        if (!SHIFTED || whole(c)) return *reinterpret_cast<const Pack<T, V> *>(row + col);
        Pack<T, V> u;
#pragma unroll
        for (int j = 0; j < V; ++j) u.e[j] = has(col, j) ? row[col + j] : from_f32<T>(0.0f);
        return u;
    }
    template <typename T> __device__ __forceinline__ void store(T *row, int c, const float (&v)[V]) const {
        const uint32_t col = first(c);
        if (!SHIFTED || whole(c)) {
            store_as<T, V>(row + col, v);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (has(col, j)) row[col + j] = from_f32<T>(v[j]);
        }
    }
    // V weights; those of SHIFTED chunks have their boundaries elsewhere.
    template <typename T> __device__ __forceinline__ void weights(const void *weight, bool f32, int c, float (&w)[V]) const {
        const uint32_t col = first(c);
        if constexpr (!SHIFTED) {
            load_weight<T, V>(weight, f32, col, w);
        } else if (!weight) {
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = 1.0f;
        } else {
            const bool all = whole(c);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float one[1] = {0.0f};
                if (all || has(col, j)) load_weight<T, 1>(weight, f32, col + j, one);
                w[j] = one[0];
            }
        }
    }
};

// The end of a row: from w s in v, the sum of s^2 and the maxima of |w s| to
// the outputs.
template <typename T, int V, int C, Scales S, bool SHIFTED>
__device__ __forceinline__ void finish_row(const NormParams &p, uint32_t row, const Chunks<V, C, SHIFTED> &chunks, float (&v)[C][V], float ss,
                                           float amax, const float (&gmax)[C], const float *group_max) {
    const float rstd = rsqrtf(ss * p.per_col + p.eps);
    // |w s| rstd rounds monotonically, so the maximum of |y| is the rounded
    // product of the maximum of |w s|.
    float scale, per_scale = 1.0f;
    if (S == kRowScale) {
        scale = scale_of(amax * rstd);
        per_scale = __fdividef(1.0f, scale);
        if (threadIdx.x == 0) p.scales[row] = scale;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t col = chunks.first(c);
        if (!chunks.some(c)) continue;
        if (S == kLaneScales || (S == kSharedScales && !SHIFTED)) {
            const uint32_t g = col >> p.group_shift;
            scale = scale_of((S == kLaneScales ? gmax[c] : group_max[g]) * rstd);
            per_scale = __fdividef(1.0f, scale);
            if (col == g << p.group_shift) p.scales[(int64_t)row * p.groups + g] = scale;
        }
        if (S == kSharedScales && SHIFTED) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (!chunks.has(col, j)) continue;
                const uint32_t g = (col + j) >> p.group_shift;
                scale = scale_of(group_max[g] * rstd);
                v[c][j] = v[c][j] * rstd * __fdividef(1.0f, scale);
                if (col + j == g << p.group_shift) p.scales[(int64_t)row * p.groups + g] = scale;
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[c][j] = S == kNoScales ? v[c][j] * rstd : v[c][j] * rstd * per_scale;
        }
        if constexpr (S == kNoScales) {
            chunks.store(static_cast<T *>(p.y) + (int64_t)row * p.cols, c, v[c]);
        } else {
            uint8_t *q = static_cast<uint8_t *>(p.y) + (int64_t)row * p.cols;
            if (!SHIFTED) {
                store_fp8<V>(q + col, v[c]);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float one[1] = {v[c][j]};
                    if (chunks.has(col, j)) store_fp8<1>(q + (col + j), one);
                }
            }
        }
    }
}

// A row (or, blockDim.y > 1, a row per warp) whose C x V values per thread
// stay in registers between the one read and the one write.  Bound by HBM,
// and by the bytes in flight that fill it: rows wait for their sums, others
// load meanwhile, so blocks an SM count.  16384 x 4096 bf16 with residual and
// e4m3 scales by 128: four blocks (51 registers) 90 us, five 82.5-84.5 us (5.6
// TB/s), six spill, 88 us; 5003 x 2049 f16 six blocks 16.4 us, five 17.4.
// The rule was chosen on these two forms.  Forms with a residual have less
// room: SHIFTED in the rows' type at six blocks and two chunks of a 16-bit type
// or four of f32 (40 registers) spill 116-128 bytes a thread, f32 of aligned
// rows at five (47-48 registers) 16-32.  There fewer blocks are better: 8192 x
// 3001 with residual, six / five / four blocks, f32 79 / 68 / 64 us, bf16 59.6 /
// 57.6 / 61.5; 16384 x 4096 f32 with residual, five / four, 164 / 161 us, to
// e4m3 by 128 148 / 131.
template <typename T, int V, int C, Scales S, bool RES, bool SHIFTED>
__global__ void __launch_bounds__(C * V >= 32 ? 512 : 256, C * V >= 32 ? 1 : SHIFTED && S == kNoScales ? 6 : 5)
norm_kernel(const __grid_constant__ NormParams p) {
    extern __shared__ float group_max[];  // kSharedScales: of each group
    __shared__ float2 red[32];
    const bool warp_rows = blockDim.y > 1;
    const uint32_t row = blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= p.rows) return;  // whole warps, which no block barrier waits for
    const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
    const T *res = RES ? static_cast<const T *>(p.residual) + row * p.residual_stride : nullptr;
    const Chunks<V, C, SHIFTED> chunks(p.cols, x, sizeof(T));
    if (S == kSharedScales) {
        for (uint32_t g = threadIdx.x; g < p.groups; g += blockDim.x) group_max[g] = 0.0f;
        __syncthreads();
    }

    Pack<T, V> ux[C], ur[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t col = chunks.first(c);
        if (chunks.some(c)) {
            ux[c] = chunks.load(x, c);
            if (RES) ur[c] = chunks.load(res, c);
        }
    }
    float v[C][V], ss = 0.0f, amax = 0.0f, gmax[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t col = chunks.first(c);
        gmax[c] = 0.0f;
        if (chunks.some(c)) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[c][j] = to_f32(ux[c].e[j]);
                if (RES) v[c][j] += to_f32(ur[c].e[j]);
                ss += v[c][j] * v[c][j];
            }
            if (RES) chunks.store(static_cast<T *>(p.sum) + (int64_t)row * p.cols, c, v[c]);
            float w[V];
            chunks.template weights<T>(p.weight, p.weight_f32, c, w);
#pragma unroll
            for (int j = 0; j < V; ++j) v[c][j] *= w[j];
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
                    const bool next = chunks.has(col, j) && (col + j) >> p.group_shift != g;
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
    finish_row<T, V, C, S, SHIFTED>(p, row, chunks, v, ss, amax, gmax, group_max);
}

// A thread's sum over a long row, up to 2^14 terms: in runs of 128, so that no
// chain of additions is longer (one chain of equal terms is off by 2e-4 there).
struct LongSum {
    float sum = 0.0f, run = 0.0f;
    uint32_t count = 0;
    __device__ __forceinline__ void add(float v) {
        run += v;
        if ((++count & 127u) == 0) {
            sum += run;
            run = 0.0f;
        }
    }
    __device__ __forceinline__ float total() const { return sum + run; }
};

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
    LongSum squares;
    float amax = 0.0f;
#pragma unroll 2
    for (uint32_t col = t * V; col < p.cols; col += blockDim.x * V) {
        float v[V], w[V], vmax = 0.0f, some = 0.0f;
        load(col, v);
        if (res) store_as<T, V>(static_cast<T *>(p.sum) + (int64_t)row * p.cols + col, v);
#pragma unroll
        for (int j = 0; j < V; ++j) some += v[j] * v[j];
        squares.add(some);
        if constexpr (FP8) {
            load_weight<T, V>(p.weight, p.weight_f32, col, w);
#pragma unroll
            for (int j = 0; j < V; ++j) vmax = fmaxf(vmax, fabsf(v[j] * w[j]));
            amax = fmaxf(amax, vmax);
            if (by_group) shared_max(&group_max[col >> p.group_shift], vmax);
        }
    }
    float ss = squares.total();
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
            const float per_scale = __fdividef(1.0f, scale);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = v[j] * rstd * per_scale;
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

// SHIFTED (see Chunks) or not: rows of whole vectors.
template <typename T, bool FP8, bool SHIFTED> heph_status launch_norm(const NormParams &p, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    constexpr int kMost = 32 / V;  // chunks of a thread: 32 registers
    const uint32_t units = SHIFTED ? (p.cols + 2 * V - 2) / V : p.cols / V;
    const size_t smem = FP8 && p.groups > 1 ? p.groups * sizeof(float) : 0;
    // Rows of up to 256 threads where the chunks reach, as rows of few warps
    // wait less for one another.
    uint32_t c = 1;
    while (c < kMost && (units + c - 1) / c > 256) c *= 2;
    const bool in_lanes = !SHIFTED && p.groups > 1 && (1u << p.group_shift) / V <= 32;
    const bool own_scales = !FP8 || p.groups == 1 || in_lanes;  // no group_max
    const uint32_t threads = ((units + c - 1) / c + 31) / 32 * 32;
    if (threads > (c * V >= 32 ? 512 : 1024)) {
        if constexpr (!SHIFTED) return launch_rows("long row norm", norm_long_kernel<T, V, FP8>, dim3(p.rows), dim3(1024), smem, stream, p);
        return launch_rows("long row norm", norm_long_kernel<T, 1, FP8>, dim3(p.rows), dim3(1024), smem, stream, p);
    }
    // Short rows: one warp each, eight to a block (not where they share group_max).
    const uint32_t per_block = threads == 32 && own_scales ? 8 : 1;
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

// Rows on their way through shared memory, kRowStages - 1 of them while one is
// worked on, so that bytes in flight cost no registers.  Each thread copies
// what it reads itself, so a copy needs no barrier but the thread's own wait.
// A part of a chunk is copied as the whole 16 bytes that it lies in (a load
// when it is read would hold up the block at every row) and masked when read.
template <int C> constexpr int kRowStages = C >= 4 ? 2 : 4;

constexpr uint32_t kDweightRun = 256;  // rows whose terms of dw are added in one chain

template <typename T, int V, int C, int OPERANDS, bool SHIFTED> struct RowRing {
    static constexpr int kStages = kRowStages<C>;
    const T *base[OPERANDS];  // null: absent
    int64_t stride[OPERANDS];
    uint32_t rows;
    const Chunks<V, C, SHIFTED> &chunks;
    Pack<T, V> *slots;  // [kStages][OPERANDS][C][threads], 16 bytes each
    uint32_t stage = 0;

    __device__ RowRing(std::initializer_list<const void *> bases, std::initializer_list<int64_t> strides, uint32_t rows_,
                       const Chunks<V, C, SHIFTED> &chunks_, void *smem)
        : rows(rows_), chunks(chunks_), slots(static_cast<Pack<T, V> *>(smem)) {
#pragma unroll
        for (int o = 0; o < OPERANDS; ++o) {
            base[o] = static_cast<const T *>(bases.begin()[o]);
            stride[o] = strides.begin()[o];
        }
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) request(blockIdx.x + i * gridDim.x, i);
    }
    __device__ __forceinline__ Pack<T, V> *slot(uint32_t at, int operand, int c) const {
        return slots + ((at * OPERANDS + operand) * C + c) * blockDim.x + threadIdx.x;
    }
    __device__ __forceinline__ void request(uint32_t row, uint32_t at) const {
        if (row < rows) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const uint32_t col = chunks.first(c);
                if (!chunks.some(c)) continue;
#pragma unroll
                for (int o = 0; o < OPERANDS; ++o)
                    if (base[o]) copy16_async(slot(at, o, c), base[o] + row * stride[o] + (int32_t)col);
            }
        }
        copies_commit();  // a group for every row, empty ones too
    }
    // The row's copies are there; a later row's go to the slot read before.
    __device__ __forceinline__ void next(uint32_t row) const {
        copies_wait<kStages - 2>();
        request(row + (kStages - 1) * gridDim.x, stage == 0 ? kStages - 1 : stage - 1);
    }
    __device__ __forceinline__ Pack<T, V> get(int operand, int c) const {
        Pack<T, V> u = *slot(stage, operand, c);
        if (SHIFTED && !chunks.whole(c)) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (!chunks.has(chunks.first(c), j)) u.e[j] = from_f32<T>(0.0f);
        }
        return u;
    }
    __device__ __forceinline__ void done() { stage = stage + 1 == kStages ? 0 : stage + 1; }
};

// The thread's weights for the same columns of every row: in registers, but
// f32 ones beside 16-bit rows, which do not fit there and are read again from L1.
template <typename T, int V, int C, bool SHIFTED> struct RowWeights {
    const void *weight;
    bool again;
    const Chunks<V, C, SHIFTED> &chunks;
    Pack<T, V> kept[C];
    __device__ RowWeights(const void *weight_, bool f32, const Chunks<V, C, SHIFTED> &chunks_)
        : weight(weight_), again(weight_ && f32), chunks(chunks_) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float w[V];
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = 1.0f;
            if (!again && chunks.some(c)) chunks.template weights<T>(weight, false, c, w);
#pragma unroll
            for (int j = 0; j < V; ++j) kept[c].e[j] = from_f32<T>(w[j]);  // exact: they are of this type
        }
    }
    __device__ __forceinline__ void get(int c, float (&w)[V]) const {
        if (again) {
            chunks.template weights<T>(weight, true, c, w);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = to_f32(kept[c].e[j]);
        }
    }
};

// Block b takes rows b, b + gridDim.x, ... (SHIFTED: gridDim.x is a multiple of V
// or covers the rows, so that all of a block's rows start the same distance
// past a boundary); its share of dw stays in registers (each thread keeps its
// columns) and goes out at the end, and before that after every kDweightRun
// rows: one chain over 2^20 rows and more is off by 1e-5 of terms that are alike.
//
// Measured at 8192 x 4096 bf16 with dsum: 104 us with rows loaded when they
// are worked on, 51-53 us through the ring (5.1-5.3 TB/s) and 5 for the sum of the
// blocks' dw; SHIFTED, without dsum: 8192 x 4095 105 us, x 8191 206; x 12000
// 154; 2^20 x 128 836 us, a row's barrier and folds for each.  (The forward norm gains
// nothing by a ring: 16384 x 4096 88 us against 90 without, narrow rows lose.)
template <typename T, int V, int C, bool SHIFTED>
__global__ void __launch_bounds__(512) norm_grad_kernel(const __grid_constant__ NormGradParams p) {
    constexpr bool kHeld = C * V <= 16;  // the row's values stay in registers between their two uses
    extern __shared__ __align__(16) unsigned char staged[];
    __shared__ float2 red[2][16];
    const Chunks<V, C, SHIFTED> chunks(p.cols, static_cast<const T *>(p.x) + blockIdx.x * p.x_stride, sizeof(T));
    const RowWeights<T, V, C, SHIFTED> weights(p.weight, p.weight_f32, chunks);
    RowRing<T, V, C, 3, SHIFTED> ring({p.x, p.dy, p.dsum}, {p.x_stride, p.dy_stride, p.dsum_stride}, p.rows, chunks, staged);
    uint32_t turn = 0;
    for (uint32_t row = blockIdx.x; row < p.rows;) {
        const bool first = row == blockIdx.x;
        const uint32_t stop = min(p.rows, row + kDweightRun * gridDim.x);
        float dw[C][V];
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < V; ++j) dw[c][j] = 0.0f;
        for (; row < stop; row += gridDim.x, turn ^= 1) {
            ring.next(row);
            float ss = 0.0f, gs = 0.0f;
            Pack<T, V> ux[kHeld ? C : 1], ug[kHeld ? C : 1];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if (chunks.some(c)) {
                    const int h = kHeld ? c : 0;
                    ux[h] = ring.get(0, c);
                    ug[h] = ring.get(1, c);
                    float w[V];
                    weights.get(c, w);
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float s = to_f32(ux[h].e[j]);
                        ss += s * s;
                        gs += to_f32(ug[h].e[j]) * w[j] * s;
                    }
                }
            }
            row_fold<true, false>(ss, gs, false, red[turn]);  // two buffers: one barrier per row is enough
            const float rstd = rsqrtf(ss * p.per_col + p.eps);
            const float along = rstd * (gs * p.per_col);  // mean(w dy xhat)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if (chunks.some(c)) {
                    const int h = kHeld ? c : 0;
                    if (!kHeld) {
                        ux[0] = ring.get(0, c);
                        ug[0] = ring.get(1, c);
                    }
                    float w[V], dx[V] = {};
                    if (p.dsum) {
                        const Pack<T, V> u = ring.get(2, c);
#pragma unroll
                        for (int j = 0; j < V; ++j) dx[j] = to_f32(u.e[j]);
                    }
                    weights.get(c, w);
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float xhat = to_f32(ux[h].e[j]) * rstd, g = to_f32(ug[h].e[j]);
                        dw[c][j] += g * xhat;
                        dx[j] += rstd * (g * w[j] - xhat * along);
                    }
                    chunks.store(static_cast<T *>(p.dx) + (int64_t)row * p.cols, c, dx);
                }
            }
            ring.done();
        }
        if (!p.partials) continue;
        float *mine = p.partials + (int64_t)blockIdx.x * p.cols;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint32_t col = chunks.first(c);
            if (!chunks.some(c)) continue;
            if (!first) {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (chunks.has(col, j)) dw[c][j] += mine[col + j];
            }
            if constexpr (!SHIFTED) {
                store_as<float, V>(mine + col, dw[c]);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (chunks.has(col, j)) mine[col + j] = dw[c][j];
            }
        }
    }
}

// Rows too long for the registers: read twice; the block's share of dw is
// gathered in its own row of `partials`, each thread its own columns.  Blocks
// of more than kDweightRun rows gather those in a second row first (there are
// two for each block then: launch_rms_norm_backward).
template <typename T, int V> __global__ void __launch_bounds__(1024) norm_grad_long_kernel(const __grid_constant__ NormGradParams p) {
    __shared__ float2 red[2][32];
    const bool runs = p.rows > kDweightRun * (uint64_t)gridDim.x;
    float *const whole = p.partials + (int64_t)blockIdx.x * p.cols;
    float *const gather = whole + (runs ? (int64_t)gridDim.x * p.cols : 0);
    uint32_t turn = 0, done = 0;  // rows of this block that are done
    auto load = [](const void *src, int64_t at, float (&v)[V]) {
        const auto u = *reinterpret_cast<const Pack<T, V> *>(static_cast<const T *>(src) + at);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = to_f32(u.e[j]);
    };
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1, ++done) {
        const bool fresh = done % kDweightRun == 0, give = runs && (done % kDweightRun == kDweightRun - 1 || row + gridDim.x >= p.rows);
        LongSum squares, products;
        for (uint32_t col = threadIdx.x * V; col < p.cols; col += blockDim.x * V) {
            float w[V], s[V], g[V], ss = 0.0f, gs = 0.0f;
            load_weight<T, V>(p.weight, p.weight_f32, col, w);
            load(p.x, row * p.x_stride + col, s);
            load(p.dy, row * p.dy_stride + col, g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                ss += s[j] * s[j];
                gs += g[j] * w[j] * s[j];
            }
            squares.add(ss);
            products.add(gs);
        }
        float ss = squares.total(), gs = products.total();
        row_fold<true, false>(ss, gs, false, red[turn]);
        const float rstd = rsqrtf(ss * p.per_col + p.eps);
        const float along = rstd * (gs * p.per_col);  // mean(w dy xhat)
        for (uint32_t col = threadIdx.x * V; col < p.cols; col += blockDim.x * V) {
            float w[V], s[V], g[V], dx[V] = {};
            load_weight<T, V>(p.weight, p.weight_f32, col, w);
            load(p.x, row * p.x_stride + col, s);
            load(p.dy, row * p.dy_stride + col, g);
            if (p.dsum) load(p.dsum, row * p.dsum_stride + col, dx);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xhat = s[j] * rstd;
                dx[j] += rstd * (g[j] * w[j] - xhat * along);
                if (!p.partials) continue;
                const float run = (fresh ? 0.0f : gather[col + j]) + g[j] * xhat;
                if (give) whole[col + j] = (done < kDweightRun ? 0.0f : whole[col + j]) + run;
                else gather[col + j] = run;
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

constexpr uint32_t kMaxRingSmem = 220 * 1024;  // of a block, and of an SM's blocks
// Blocks an SM of the gradient's kernel: about 24 warps, as many as its
// registers and its ring let run at once.  A narrow row has few of them.
uint32_t grad_blocks_per_sm(uint32_t threads, size_t smem) {
    return std::clamp(std::min(768 / threads, kMaxRingSmem / (uint32_t)smem), 1u, 4u);
}

template <typename T, int V, bool SHIFTED>
heph_status launch_norm_grad(const NormGradParams &p, uint32_t partials, int sm_count, uint32_t *out_blocks, cudaStream_t stream) {
    constexpr int kMost = 32 / V;  // chunks of a thread: 32 registers of dw
    const uint32_t units = SHIFTED ? (p.cols + 2 * V - 2) / V : p.cols / V;
    uint32_t c = 1;
    while (c < kMost && (units + c - 1) / c > (c * V >= 16 ? 512 : 256)) c *= 2;
    const uint32_t threads = ((units + c - 1) / c + 31) / 32 * 32;
    const size_t smem = (size_t)(c >= 4 ? kRowStages<4> : kRowStages<1>) * 3 * 16 * c * threads;
    if (threads > 512 || smem > kMaxRingSmem) {
        *out_blocks = std::min<uint32_t>(partials, sm_count);
        if constexpr (!SHIFTED)
            return launch_rows("long row norm gradient", norm_grad_long_kernel<T, V>, dim3(*out_blocks), dim3(1024), 0, stream, p);
        return launch_rows("long row norm gradient", norm_grad_long_kernel<T, 1>, dim3(*out_blocks), dim3(1024), 0, stream, p);
    }
    auto go = [&]<int C>() -> heph_status {
        auto kernel = norm_grad_kernel<T, V, C, SHIFTED>;
        const uint32_t step = SHIFTED ? V : 1, most = grad_blocks_per_sm(threads, smem) * sm_count / step * step;
        *out_blocks = std::min(partials, most);
        HEPH_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxRingSmem),
                      HEPH_DISPATCH_FAILED, "row norm gradient shared memory");
        return launch_rows("row norm gradient", kernel, dim3(*out_blocks), dim3(threads), smem, stream, p);
    };
    if (c == 1) return go.template operator()<1>();
    if (c == 2) return go.template operator()<2>();
    if (c == 4) return go.template operator()<4>();
    if constexpr (kMost >= 8) return go.template operator()<8>();
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

// The most blocks that launch_norm_grad starts (4 an SM for rows of up to 192
// threads, else 3), in whole vectors' worth.  norm_grad_long_kernel, of one
// block an SM, has two rows of partials for each where the blocks have more rows than one.
uint32_t norm_grad_partials(uint32_t rows, uint32_t cols, int sm_count) {
    const uint32_t most = (cols <= 3000 ? 4 : 3) * (uint32_t)sm_count;
    return rows < most ? rows : most / 8 * 8;
}

heph_status launch_rms_norm_backward(const NormGradArgs &a, int sm_count, cudaStream_t stream) {
    const uint32_t partials = norm_grad_partials(a.rows, a.cols, sm_count);
    uint32_t blocks = 0;  // of these used
    const NormGradParams p{a.dy.ptr, a.x.ptr, a.dsum.ptr, a.weight, a.dx, a.dweight ? a.partials : nullptr, a.dy.stride,
                           a.x.stride, a.dsum.stride, a.eps, 1.0f / a.cols, a.rows, a.cols, a.weight_f32};
    return dispatch_row_dtype(a.dtype, [&]<typename T>() {
        constexpr int V = 16 / sizeof(T);
        if (a.rows) {
            const bool wide = a.cols % V == 0 && aligned_rows(a.dy, sizeof(T)) && aligned_rows(a.x, sizeof(T)) &&
                              aligned_rows(a.dsum, sizeof(T)) && aligned16(a.weight) && aligned16(a.dx);
            // Shifted rows, as in launch_rms_norm; else element by element.
            auto like = [&](const void *ptr, int64_t stride) {
                const auto apart = reinterpret_cast<intptr_t>(ptr) - reinterpret_cast<intptr_t>(a.x.ptr);
                return !ptr || (apart % 16 == 0 && (stride - a.x.stride) % V == 0);
            };
            const bool shifted = like(a.dy.ptr, a.dy.stride) && like(a.dsum.ptr, a.dsum.stride) && like(a.dx, a.cols);
            heph_status st;
            if (wide) {
                st = launch_norm_grad<T, V, false>(p, partials, sm_count, &blocks, stream);
            } else if (shifted) {
                st = launch_norm_grad<T, V, true>(p, partials, sm_count, &blocks, stream);
            } else {
                blocks = std::min<uint32_t>(partials, sm_count);
                st = launch_rows("row norm gradient", norm_grad_long_kernel<T, 1>, dim3(blocks), dim3(1024), 0, stream, p);
            }
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
