// expert_route.cu — routing of tokens to experts, and its gradient.
//
//   s = softmax(l) or sigmoid(l);  c = s + bias chooses, s weighs
//   groups: a group counts as the sum of its one or two best c; the best
//   `groups_kept` groups stay.  The k experts of largest c (without a bias: of
//   largest l, which is the same order), lowest index first among equals.
//   w_j = scale s_j, or renormalised scale s_j / sum of the chosen s
//
// An expert of logit (or bias) -inf or NaN is not chosen; where fewer than k are left,
// the rest of the row is -1 with weight 0.
#include "row_ops.h"
#include "row_utils.cuh"

namespace heph {

namespace {

constexpr int kRouteWarps = 4;

struct RouteParams {
    const void *logits;
    const float *bias;
    int64_t stride;
    uint32_t rows, experts, k, groups, groups_kept;
    uint32_t group_size, group_lanes, group_shift;  // lanes = 2^shift; 0 where a group is not a power of two of lanes
    bool sigmoid, renormalize, top2;
    float scale;
    float *weights;
    int32_t *picks;
};

// exp(l - m) with m the row's maximum; an infinite maximum shares all weight.
__device__ __forceinline__ float exp_below(float l, float m) { return l == m ? 1.0f : expf(l - m); }

// Weight of the row's lane-th choice (logit l, chosen or not).  m, z: maximum
// and sum of exp(l - m) over the row, of a softmax that is not renormalised.
__device__ __forceinline__ float choice_weight(float l, bool chosen, bool sigmoid, bool renormalize, float m, float z) {
    if (!renormalize) return !chosen ? 0.0f : sigmoid ? 1.0f / (1.0f + expf(-l)) : __fdividef(exp_below(l, m), z);
    // Ratios of scores need no row sum, and hold where every score underflows:
    // sigmoid(l) = exp(min(l, 0)) / (1 + exp(-|l|)).
    const float top = key_value(__reduce_max_sync(kFullMask, chosen ? ordered_number(l) : ordered_number(-INFINITY)));
    float s = 0.0f;
    if (chosen) s = sigmoid ? __fdividef(expf(fminf(l, 0.0f) - fminf(top, 0.0f)), 1.0f + expf(-fabsf(l))) : exp_below(l, top);
    const float sum = warp_sum(s);
    return sum > 0.0f ? __fdividef(s, sum) : 0.0f;
}

// N adjacent elements of a row from element `e` on; those past `end` are -inf.
// N elements of 16-byte pieces in one go where the row allows it.
template <typename T, int N> __device__ __forceinline__ void load_run(const T *src, uint32_t e, uint32_t end, float (&v)[N]) {
    constexpr int P = N * sizeof(T) < 16 ? N : 16 / sizeof(T);
    if (e + N <= end && (reinterpret_cast<uintptr_t>(src + e) & (P * sizeof(T) - 1)) == 0) {
#pragma unroll
        for (int i = 0; i < N; i += P) {
            const auto u = *reinterpret_cast<const Pack<T, P> *>(src + e + i);
#pragma unroll
            for (int j = 0; j < P; ++j) v[i + j] = to_f32(u.e[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = e + j < end ? to_f32(src[e + j]) : -INFINITY;
    }
}

template <typename T, int N> __device__ __forceinline__ void store_run(T *dst, uint32_t e, uint32_t end, const float (&v)[N]) {
    constexpr int P = N * sizeof(T) < 16 ? N : 16 / sizeof(T);
    if (e + N <= end && (reinterpret_cast<uintptr_t>(dst + e) & (P * sizeof(T) - 1)) == 0) {
#pragma unroll
        for (int i = 0; i < N; i += P) {
            Pack<T, P> u;
#pragma unroll
            for (int j = 0; j < P; ++j) u.e[j] = from_f32<T>(v[i + j]);
            *reinterpret_cast<Pack<T, P> *>(dst + e + i) = u;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (e + j < end) dst[e + j] = from_f32<T>(v[j]);
    }
}

// 1 / (1 + exp(-l)) and exp(x) for the choice, to the bounds at `off` below.
__device__ __forceinline__ float fast_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float fast_exp(float x) { return fast_exp2(x * 1.4426950408889634f); }
__device__ __forceinline__ float fast_sigmoid(float l) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + fast_exp(-l)));
    return r;
}

// Whether the values of the groups that stay and of those that go (by lane) are
// further apart than what 32 bits may be off by: `least` for their scores, and
// roundings of their sums of |c| size_of.
__device__ __forceinline__ bool groups_apart(float value, float size_of, bool stays, bool is_group, float least) {
    const uint32_t key = ordered_number(value);
    const uint32_t low = __reduce_min_sync(kFullMask, stays ? key : ~0u);
    const uint32_t high = __reduce_max_sync(kFullMask, !stays && is_group ? key : 0u);
    const float size = __uint_as_float(__reduce_max_sync(kFullMask, is_group ? __float_as_uint(size_of) : 0u));
    // -inf is exact: a group with nothing to choose.
    return !high || !(key_value(low) - key_value(high) <= least + 0x1p-22f * size);
}

// score + bias of the row's experts in 64 bits, lane i's N from i N on; -inf
// where an expert may not be chosen.  Written out once (unroll 1): few rows
// come here, and what they wait for is mostly instructions.
template <typename T, int N>
__device__ __forceinline__ void exact_values(const RouteParams &p, const T *src, float m, double (&c)[N]) {
    const uint32_t lane = threadIdx.x & 31;
    double total = 0.0;
#pragma unroll 1
    for (int j = 0; j < N; ++j) {
        const uint32_t e = lane * N + j;
        const float l = e < p.experts ? to_f32(src[e]) : -INFINITY;
        const double x = exp(p.sigmoid ? -(double)l : l == m ? 0.0 : (double)l - (double)m);
        c[j] = !(l > -INFINITY) ? -INFINITY : p.sigmoid ? 1.0 / (1.0 + x) : x;
        if (!p.sigmoid && l > -INFINITY) total += x;
    }
    if (!p.sigmoid) total = warp_fold<double, OP_SUM>(total);
#pragma unroll 1
    for (int j = 0; j < N; ++j) {
        const uint32_t e = lane * N + j;
        if (!(c[j] > -INFINITY)) continue;
        if (!p.sigmoid) c[j] /= total;
        if (p.bias) c[j] += p.bias[e];
        if (!(c[j] > -INFINITY)) c[j] = -INFINITY;
    }
}

// The groups that stay, a bit each, in 64 bits.
template <typename T, int N> __device__ __noinline__ uint32_t exact_groups(const RouteParams &p, const T *src, float m) {
    const uint32_t lane = threadIdx.x & 31;
    double c[N], mine = -INFINITY;  // of lane g: the value of group g
    exact_values<T, N>(p, src, m, c);
#pragma unroll 1
    for (uint32_t g = 0; g < p.groups; ++g) {
        const uint32_t begin = g * p.group_size;
        double a = -INFINITY, b = -INFINITY;  // best and second
        if (lane * N + N > begin && lane * N < begin + p.group_size) {
#pragma unroll 1
            for (int j = 0; j < N; ++j) {
                if (lane * N + j < begin || lane * N + j >= begin + p.group_size) continue;
                b = fmax(b, fmin(a, c[j]));
                a = fmax(a, c[j]);
            }
        }
#pragma unroll 1
        for (int d = 16; d > 0; d >>= 1) {
            const double oa = shfl_xor(a, d), ob = shfl_xor(b, d);
            b = fmax(fmax(b, ob), fmin(a, oa));
            a = fmax(a, oa);
        }
        if (p.top2 && b > -INFINITY) a += b;
        if (lane == g) mine = a;
    }
    uint32_t ahead = 0;
    for (uint32_t g = 0; g < p.groups; ++g) {
        const double o = shfl_idx(mine, g);
        ahead += o > mine || (o == mine && g < lane);
    }
    return __ballot_sync(kFullMask, lane < p.groups && ahead < p.groups_kept);
}

// Lane i's choice in 64 bits, for rows of more near candidates than lanes;
// `kept`: the groups that stay.
template <typename T, int N> __device__ __noinline__ int32_t exact_choice(const RouteParams &p, const T *src, float m, uint32_t kept) {
    const uint32_t lane = threadIdx.x & 31;
    double c[N];
    if (p.bias) {
        exact_values<T, N>(p, src, m, c);
    } else {
        for (int j = 0; j < N; ++j) {
            const float l = lane * N + j < p.experts ? to_f32(src[lane * N + j]) : -INFINITY;
            c[j] = l == l ? l : -INFINITY;
        }
    }
    for (int j = 0; j < N; ++j)
        if (p.groups > 1 && lane * N + j < p.experts && !(kept >> ((lane * N + j) / p.group_size) & 1u)) c[j] = -INFINITY;
    int32_t pick = -1;
#pragma unroll 1
    for (uint32_t i = 0; i < p.k; ++i) {
        double best = -INFINITY;
        uint32_t at = 0xffffffffu;
#pragma unroll 1
        for (int j = 0; j < N; ++j) {
            if (c[j] > best) {
                best = c[j];
                at = lane * N + j;
            }
        }
        warp_arg_fold<double, OP_MAX>(best, at);
        if (at == 0xffffffffu) break;  // nothing left, for every lane
        if (at / N == lane) c[at % N] = -INFINITY;
        if (lane == i) pick = (int32_t)at;
    }
    return pick;
}

// The rank of candidate `mine` (of the first `count` lanes, one each) by the
// 64-bit values of score + bias or of the logits, equal ones by expert.
template <typename T, int N>
__device__ __noinline__ void exact_rank(const RouteParams &p, const T *src, uint32_t mine, uint32_t lane, uint32_t count, float m,
                                        double *values, const uint2 *candidates, uint32_t &rank) {
    const uint32_t lanes = (uint32_t)((1ull << count) - 1);
    const float l = to_f32(src[mine]);
    double c = l;
    if (p.bias) {
        if (p.sigmoid) {
            c = 1.0 / (1.0 + exp(-c));
        } else {
            double z = 0.0;  // of the row, the experts dealt to the lanes
            for (uint32_t e = lane; e < p.experts; e += count) {
                const float o = to_f32(src[e]);
                z += o == m ? 1.0 : o > -INFINITY ? exp((double)o - (double)m) : 0.0;
            }
            values[lane] = z;
            __syncwarp(lanes);
            z = 0.0;
            for (uint32_t i = 0; i < count; ++i) z += values[i];
            __syncwarp(lanes);
            c = (l == m ? 1.0 : exp(c - (double)m)) / z;
        }
        c += p.bias[mine];
    }
    values[lane] = c;
    __syncwarp(lanes);
    rank = 0;
    for (uint32_t i = 0; i < count; ++i) rank += values[i] > c || (values[i] == c && candidates[i].y < mine);
    __syncwarp(lanes);
}

// Sorts N values a lane into falling order (Batcher's odd-even merges).
template <int N> __device__ __forceinline__ void sort_falling(uint32_t (&v)[N]) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const uint32_t a = v[i + j], b = v[i + j + k];
                        v[i + j] = max(a, b);
                        v[i + j + k] = min(a, b);
                    }
}

// Bound by instruction issue: 32768 x 256 f32, sigmoid, bias, 8 groups, takes
// 35-43 us (by how many rows 64 bits decide) with 79 % of the issue slots filled
// and the ALU pipe 71 % busy, 900 warp instructions a row, of which the sort is 38
// minima and maxima; without groups 26 (softmax) and 30 us (sigmoid, bias), 32768 x
// 64 19 us.
//
// A warp per row, lane i holds experts i N ... i N + N - 1.  The choice is
// made in 32 bits and checked: where a gap that decides something is not
// wider than what 32 bits may be off by, 64 bits decide: of the candidates
// (about 2 rows in 1000 with a sigmoid and a bias), or, where the groups are
// in doubt (1 in 30000), of the whole row.
template <typename T, int N> __global__ void __launch_bounds__(32 * kRouteWarps, N <= 8 ? 10 : 1)
route_kernel(const __grid_constant__ RouteParams p) {
    constexpr uint32_t kLow = N - 1;  // the low bits of a key hold N - 1 - j
    const uint32_t lane = threadIdx.x & 31, row = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    const T *src = static_cast<const T *>(p.logits) + row * p.stride;
    float c[N], m = 0.0f, z = 1.0f;
    load_run<T, N>(src, lane * N, p.experts, c);
    if (!p.sigmoid && (p.bias || p.groups > 1 || !p.renormalize)) {
        m = -INFINITY;
#pragma unroll
        for (int j = 0; j < N; ++j) m = fmaxf(m, c[j]);
        m = warp_max(m);
        z = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j)
            z += !(c[j] > -INFINITY) ? 0.0f : c[j] == m ? 1.0f : p.renormalize ? fast_exp(c[j] - m) : expf(c[j] - m);
        z = warp_sum(z);
    }
    // What a score may be off by.  Sigmoid: a quarter of the exp's error (a
    // unit and a half, and its rounded exponent l with |l| s (1 - s) < 1/4),
    // half a unit of the sum and a unit of the reciprocal, below 2^-22.  Softmax: those, ten levels of the sum, whose
    // terms' exponents average below ln 1024, and the quotient, below 2^-18.
    const float score_off = p.sigmoid ? 0x1p-22f : 0x1p-18f;
    const float inverse = 1.0f / z;
    auto score = [&](float l) { return p.sigmoid ? fast_sigmoid(l) : l == m ? inverse : fast_exp(l - m) * inverse; };
    // A key in the order of the choice: of score + bias, or of the logit; 0
    // is not to be chosen.  Its low bits say which of the lane's it is.
    auto key_of = [&](float v, int j) { return v > -INFINITY ? (ordered_number(v) & ~kLow) | (kLow - j) : 0u; };
    uint32_t key[N];
    if (p.bias) {
        float b[N];
        load_run<float, N>(p.bias, lane * N, p.experts, b);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            c[j] = c[j] > -INFINITY ? score(c[j]) + b[j] : -INFINITY;
            key[j] = key_of(c[j], j);
            if (!key[j]) c[j] = -INFINITY;  // a NaN bias: no minimum or maximum passes over it both ways
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            key[j] = key_of(c[j], j);
            if (!key[j]) c[j] = -INFINITY;
        }
    }
    // Half of what two keys' values may differ by and yet be in the other
    // order: the score's error, a rounding of the sum, a unit of the last kept bit.
    const float key_off = p.bias ? score_off : 0.0f;
    constexpr float kKeyStep = 0x1p-23f * (N + 1);
    uint32_t kept = 0;  // the groups that stay, a bit each
    if (p.groups > 1 && !p.group_lanes) {
        // Groups of any size: each group's best two of all lanes, in turn.
        float mine = -INFINITY, size_of = 0.0f;  // lane g: the value of group g
        for (uint32_t g = 0; g < p.groups; ++g) {
            float a = -INFINITY, b = -INFINITY;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t e = lane * N + j;
                if (key[j] && e >= g * p.group_size && e - g * p.group_size < p.group_size) {
                    const float v = p.bias ? c[j] : score(c[j]);
                    b = fmaxf(b, fminf(a, v));
                    a = fmaxf(a, v);
                }
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) {
                const float oa = shfl_xor(a, d), ob = shfl_xor(b, d);
                b = fmaxf(fmaxf(b, ob), fminf(a, oa));
                a = fmaxf(a, oa);
            }
            if (!p.top2 || !(b > -INFINITY)) b = 0.0f;
            if (lane == g) {
                mine = a + b;
                size_of = mine > -INFINITY ? fabsf(a) + fabsf(b) : 0.0f;
            }
        }
        uint32_t ahead = 0;
        for (uint32_t g = 0; g < p.groups; ++g) {
            const float o = shfl_idx(mine, g);
            ahead += o > mine || (o == mine && g < lane);
        }
        const bool stays = lane < p.groups && ahead < p.groups_kept;
        kept = groups_apart(mine, size_of, stays, lane < p.groups, 4.0f * score_off)
                   ? __ballot_sync(kFullMask, stays)
                   : exact_groups<T, N>(p, src, m);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t e = lane * N + j;
            if (e < p.experts && !(kept >> (e / p.group_size) & 1u)) key[j] = 0;
        }
    }
    // Best and second of the lane's experts, to value its group by: of score +
    // bias, or of the logits, whose order is the scores'.  (Not of the keys,
    // whose low bits are not the value's.)
    float best = -INFINITY, second = -INFINITY;
    if (p.group_lanes && p.groups > 1) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            second = fmaxf(second, fminf(best, c[j]));
            best = fmaxf(best, c[j]);
        }
    }
    sort_falling<N>(key);  // each lane's; the row's next is the largest head
    if (p.groups > 1 && p.group_lanes) {
        // A group is a power of two of whole lanes, which share the comparisons.
        float a = best, b = second;
        if (!p.bias) {
            a = best > -INFINITY ? score(best) : -INFINITY;
            b = second > -INFINITY ? score(second) : -INFINITY;
        }
        for (uint32_t d = 1; d < p.group_lanes; d *= 2) {
            const float oa = shfl_xor(a, d), ob = shfl_xor(b, d);
            b = fmaxf(fmaxf(b, ob), fminf(a, oa));
            a = fmaxf(a, oa);
        }
        if (!p.top2 || !(b > -INFINITY)) b = 0.0f;
        const float mine = a + b, size_of = mine > -INFINITY ? fabsf(a) + fabsf(b) : 0.0f;
        const uint32_t own = lane >> p.group_shift, share = lane & (p.group_lanes - 1);
        uint32_t ahead = 0;
        for (uint32_t g = share; g < p.groups + share; g += p.group_lanes) {
            const uint32_t from = g << p.group_shift;
            const float o = __shfl_sync(kFullMask, mine, from);
            if (g < p.groups) ahead += o > mine || (o == mine && g < own);
        }
        for (uint32_t d = 1; d < p.group_lanes; d *= 2) ahead += __shfl_xor_sync(kFullMask, ahead, d);
        bool stays = own < p.groups && ahead < p.groups_kept;
        if (groups_apart(mine, size_of, stays, own < p.groups, 4.0f * score_off)) {
            kept = __reduce_or_sync(kFullMask, stays ? 1u << own : 0u);
        } else {
            kept = exact_groups<T, N>(p, src, m);
            stays = own < p.groups && (kept >> own & 1u);
        }
        if (!stays) {
#pragma unroll
            for (int j = 0; j < N; ++j) key[j] = 0;
        }
    }
    // The row's first k, and one more to check the last by: of lane i the
    // i-th key, its low bits cleared, and its expert.  Key 0: none is left.
    __shared__ uint2 listed[kRouteWarps][32], winners[kRouteWarps][32];
    __shared__ double values[kRouteWarps][32];
    uint2 *candidates = listed[threadIdx.x >> 5], *won_by = winners[threadIdx.x >> 5];
    const uint32_t turns = min(p.k + 1, 32u), lower = (1u << lane) - 1;
    won_by[lane] = make_uint2(0, 0);
    auto entry = [&](uint32_t k) { return make_uint2(k & ~kLow, lane * N + kLow - (k & kLow)); };
    // k + 1 lanes have a key at or above the (k+1)-th largest head: the
    // candidates are the keys that reach it, few more than k + 1.
    // (And the keys that are less than the margin below it, which 64 bits may
    // place before it.)
    auto margin = [&](float v) { return 2.0f * (key_off + fabsf(v) * kKeyStep) + 0x1p-120f; };
    // Keys of 16-bit logits themselves lose nothing in the low bits: equal
    // keys are equal logits, which the index settles.
    const bool exact = !p.bias && sizeof(T) == 2;
    uint32_t least = 1, count = 0;
    if (turns <= 13) {
        uint32_t head = key[0] & ~kLow;
        for (uint32_t i = 0; i < turns; ++i) {
            least = __reduce_max_sync(kFullMask, head);
            if (head == least) head = 0;
        }
        const float bound = key_value(least) - 2.0f * margin(key_value(least));
        if (least && !exact && bound == bound) least = ordered_number(bound) & ~kLow;  // (+inf is its own bound)
        least = max(least, 1u);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t reach = __ballot_sync(kFullMask, (key[j] & ~kLow) >= least);
            if (!reach) break;
            const uint32_t at = count + __popc(reach & lower);
            if ((reach >> lane & 1u) && at < 32) candidates[at] = entry(key[j]);
            count += __popc(reach);
        }
    } else {
        count = 33;
    }
    __syncwarp();
    if (count <= 32) {
        // Each lane ranks one of them; equal keys by expert.
        const uint2 mine = lane < count ? candidates[lane] : make_uint2(0, 0);
        uint32_t rank = 0;
        for (uint32_t i = 0; i < count; ++i) {
            const uint2 o = candidates[i];
            rank += o.x > mine.x || (o.x == mine.x && o.y < mine.y);
        }
        if (lane < count) won_by[rank] = mine;
        __syncwarp();
        if (!exact) {
            const uint32_t next = lane < 31 ? won_by[lane + 1].x : 0;
            const float a = key_value(won_by[lane].x);
            const bool near = lane < p.k && next && a - key_value(next) <= margin(a);
            if (__any_sync(kFullMask, near)) {
                // Ranks by the 64-bit values of the candidates.
                __syncwarp();
                if (lane < count) {
                    exact_rank<T, N>(p, src, mine.y, lane, count, m, values[threadIdx.x >> 5], candidates, rank);
                    won_by[rank] = mine;
                }
            }
        }
    } else {
        // Many to choose, or few lanes to choose from: one after the other.
        for (uint32_t i = 0; i < turns; ++i) {
            const uint32_t head = key[0] & ~kLow;
            const uint32_t best = __reduce_max_sync(kFullMask, head);
            const uint32_t owners = __ballot_sync(kFullMask, head == best);
            if (best && head == best && !(owners & lower)) {  // the lowest of them
                won_by[i] = entry(key[0]);
#pragma unroll
                for (int j = 0; j + 1 < N; ++j) key[j] = key[j + 1];
                key[N - 1] = 0;
            }
        }
    }
    __syncwarp();
    const uint2 won = won_by[lane];
    bool sure = true;
    if (count > 32 && !exact && lane < p.k && won.x) {
        const uint32_t next = lane < 31 ? won_by[lane + 1].x : 0;
        const float a = key_value(won.x);
        if (next && a - key_value(next) <= margin(a)) sure = false;
        if (p.k == 32) sure = false;  // there is no lane for the 33rd
    }
    int32_t pick = won.x && lane < p.k ? (int32_t)won.y : -1;
    if (!__all_sync(kFullMask, sure)) pick = exact_choice<T, N>(p, src, m, kept);
    const float logit = pick >= 0 ? to_f32(src[pick]) : 0.0f;
    const float w = choice_weight(logit, pick >= 0, p.sigmoid, p.renormalize, m, z);
    if (lane < p.k) {
        p.weights[(int64_t)row * p.k + lane] = w * p.scale;
        p.picks[(int64_t)row * p.k + lane] = pick;
    }
}

struct RouteGradParams {
    const void *logits;
    const float *dweights;
    const int32_t *picks;
    int64_t stride, dweights_stride, picks_stride;
    uint32_t rows, experts, k;
    bool sigmoid, renormalize;
    float scale;
    void *dlogits;
};

// Renormalised, with r = w / scale:  d(log s_j) = scale r_j (g_j - sum g r),
// else d(log s_j) = scale s_j g_j;  then for a sigmoid dl_j = d(log s_j)
// (1 - s_j), for a softmax dl_i = d(log s_i) - s_i sum of all d(log s), whose
// last term vanishes when renormalised.
template <typename T, int N> __global__ void __launch_bounds__(32 * kRouteWarps)
route_grad_kernel(const __grid_constant__ RouteGradParams p) {
    // The row's gradient of the log scores, by expert; first used to see
    // whether an expert is named twice.
    __shared__ __align__(16) float by_expert[kRouteWarps][32 * N];
    const uint32_t lane = threadIdx.x & 31, row = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    const T *src = static_cast<const T *>(p.logits) + row * p.stride;
    float *at = by_expert[threadIdx.x >> 5];
    using Run = Pack<float, N < 4 ? N : 4>;
    Run *own = reinterpret_cast<Run *>(at + lane * N);
    constexpr int kRuns = N < 4 ? 1 : N / 4;
#pragma unroll
    for (int i = 0; i < kRuns; ++i) own[i] = Run{};
    uint32_t pick = ~0u;
    float logit = 0.0f, g = 0.0f;
    if (lane < p.k) {
        pick = (uint32_t)p.picks[row * p.picks_stride + lane];
        if (pick < p.experts) {
            g = p.dweights[row * p.dweights_stride + lane];
            logit = to_f32(src[pick]);
        }
    }
    const bool whole = !p.sigmoid && !p.renormalize;  // every logit has a gradient
    float l[N], m = -INFINITY, z = 0.0f;
    if (whole) {
        load_run<T, N>(src, lane * N, p.experts, l);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (!(l[j] == l[j])) l[j] = -INFINITY;
            m = fmaxf(m, l[j]);
        }
        m = key_value(__reduce_max_sync(kFullMask, ordered_number(m)));
#pragma unroll
        for (int j = 0; j < N; ++j) {
            l[j] = l[j] == m ? 1.0f : fast_exp(l[j] - m);
            z += l[j];
        }
        z = m > -INFINITY ? warp_sum(z) : 0.0f;
    }
    const bool chosen = pick < p.experts && logit > -INFINITY;
    if (!chosen) g = 0.0f;
    const float r = choice_weight(logit, chosen, p.sigmoid, p.renormalize, m, z);
    const float dot = warp_sum(g * r);
    float d = p.scale * r * (p.renormalize ? g - dot : g);
    if (p.sigmoid) d /= 1.0f + expf(logit);
    __syncwarp();
    if (chosen) at[pick] = __uint_as_float(lane);
    __syncwarp();
    const bool alone = !chosen || at[pick] == __uint_as_float(lane);
    __syncwarp();
    if (__all_sync(kFullMask, alone)) {
        if (chosen) at[pick] = d;
    } else {
        // In turn, so that the sum of an expert's does not depend on an order.
        if (chosen) at[pick] = 0.0f;
        for (uint32_t i = 0; i < p.k; ++i) {
            __syncwarp();
            if (lane == i && chosen) at[pick] += d;
        }
    }
    __syncwarp();
    float dl[N];
    const float rest = whole && z > 0.0f ? -p.scale * dot / z : 0.0f;
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
        const Run u = own[i];
#pragma unroll
        for (int j = 0; j < N / kRuns; ++j) dl[i * (N / kRuns) + j] = u.e[j] + (whole ? rest * l[i * (N / kRuns) + j] : 0.0f);
    }
    store_run<T, N>(static_cast<T *>(p.dlogits) + (int64_t)row * p.experts, lane * N, p.experts, dl);
}

// Calls f.template operator()<N>() with the experts per lane.
template <typename F> heph_status dispatch_experts(uint32_t experts, F &&f) {
    if (experts <= 32) return f.template operator()<1>();
    if (experts <= 64) return f.template operator()<2>();
    if (experts <= 128) return f.template operator()<4>();
    if (experts <= 256) return f.template operator()<8>();
    if (experts <= 512) return f.template operator()<16>();
    return f.template operator()<32>();
}

}  // namespace

heph_status launch_route(const RouteArgs &a, cudaStream_t stream) {
    RouteParams p{a.logits.ptr, a.bias, a.logits.stride, a.rows, a.experts, a.k, a.groups, a.groups_kept, a.experts / a.groups,
                  0, 0, a.sigmoid, a.renormalize, a.group_top == 2, a.scale, a.weights, a.picks};
    const dim3 grid((a.rows + kRouteWarps - 1) / kRouteWarps);
    return dispatch_row_dtype(a.dtype, [&]<typename T>() {
        return dispatch_experts(a.experts, [&]<int N>() {
            const uint32_t lanes = p.group_size / N;
            if (p.group_size % N == 0 && (lanes & (lanes - 1)) == 0) {
                p.group_lanes = lanes;
                p.group_shift = __builtin_ctz(lanes);
            }
            return launch_rows("expert routing", route_kernel<T, N>, grid, dim3(32 * kRouteWarps), 0, stream, p);
        });
    });
}

heph_status launch_route_backward(const RouteGradArgs &a, cudaStream_t stream) {
    const RouteGradParams p{a.logits.ptr, static_cast<const float *>(a.dweights.ptr), static_cast<const int32_t *>(a.picks.ptr),
                            a.logits.stride, a.dweights.stride, a.picks.stride, a.rows, a.experts, a.k,
                            a.sigmoid, a.renormalize, a.scale, a.dlogits};
    const dim3 grid((a.rows + kRouteWarps - 1) / kRouteWarps);
    return dispatch_row_dtype(a.dtype, [&]<typename T>() {
        return dispatch_experts(a.experts, [&]<int N>() {
            return launch_rows("expert routing gradient", route_grad_kernel<T, N>, grid, dim3(32 * kRouteWarps), 0, stream, p);
        });
    });
}

}  // namespace heph
