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
    if (!renormalize) return !chosen ? 0.0f : sigmoid ? 1.0f / (1.0f + expf(-l)) : exp_below(l, m) / z;
    // Ratios of scores need no row sum, and hold where every score underflows:
    // sigmoid(l) = exp(min(l, 0)) / (1 + exp(-|l|)).
    const float top = key_value(__reduce_max_sync(kFullMask, chosen ? ordered_number(l) : ordered_number(-INFINITY)));
    float s = 0.0f;
    if (chosen) s = sigmoid ? expf(fminf(l, 0.0f) - fminf(top, 0.0f)) / (1.0f + expf(-fabsf(l))) : exp_below(l, top);
    const float sum = warp_sum(s);
    return sum > 0.0f ? s / sum : 0.0f;
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

// The choice in 64 bits, for rows where 32 leave it open: a warp per row, lane
// i holds experts i N ... i N + N - 1.
template <typename T, int N> __device__ __noinline__ int32_t choose_exactly(const RouteParams &p, const T *src) {
    const uint32_t lane = threadIdx.x & 31;
    float l[N], m = -INFINITY;
    load_run<T, N>(src, lane * N, p.experts, l);
    uint32_t open = 0;  // experts that may still be chosen, a bit per j
    double c[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if (!(l[j] == l[j])) l[j] = -INFINITY;
        m = fmaxf(m, l[j]);
        open |= (l[j] > -INFINITY ? 1u : 0u) << j;
        c[j] = l[j];
    }
    m = warp_max(m);
    if (p.bias || p.groups > 1) {
        double total = 0.0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const double d = l[j];
            if (p.sigmoid) c[j] = 1.0 / (1.0 + exp(-d));
            else c[j] = !(open >> j & 1u) ? 0.0 : l[j] == m ? 1.0 : exp(d - m);
            total += c[j];
        }
        if (!p.sigmoid) {
            total = warp_fold<double, OP_SUM>(total);
#pragma unroll
            for (int j = 0; j < N; ++j) c[j] /= total;
        }
        if (p.bias) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t e = lane * N + j;
                if (e < p.experts) c[j] += p.bias[e];
                if (!(c[j] > -INFINITY)) open &= ~(1u << j);
            }
        }
        if (p.groups > 1) {
            const uint32_t size = p.group_size;
            double mine = -INFINITY;  // lane g: the value of group g
            for (uint32_t g = 0; g < p.groups; ++g) {
                double a = -INFINITY, b = -INFINITY;  // best and second
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const uint32_t e = lane * N + j;
                    if ((open >> j & 1u) && e >= g * size && e - g * size < size) {
                        b = fmax(b, fmin(a, c[j]));
                        a = fmax(a, c[j]);
                    }
                }
#pragma unroll
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
            const uint32_t kept = __ballot_sync(kFullMask, lane < p.groups && ahead < p.groups_kept);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t e = lane * N + j;
                if (e < p.experts && !(kept >> (e / size) & 1u)) open &= ~(1u << j);
            }
            if (!p.bias) {
#pragma unroll
                for (int j = 0; j < N; ++j) c[j] = l[j];
            }
        }
    }
    int32_t pick = -1;
    for (uint32_t i = 0; i < p.k; ++i) {
        double best = -INFINITY;
        uint32_t at = 0xffffffffu;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if ((open >> j & 1u) && (at == 0xffffffffu || c[j] > best)) {
                best = c[j];
                at = lane * N + j;
            }
        }
        warp_arg_fold<double, OP_MAX>(best, at);
        if (at == 0xffffffffu) break;  // nothing left, for every lane
        if (at / N == lane) open &= ~(1u << (at % N));
        if (lane == i) pick = (int32_t)at;
    }
    return pick;
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

// A warp per row, lane i holds experts i N ... i N + N - 1.  The choice is
// made in 32 bits and checked: where a gap that decides something is not
// wider than what 32 bits may be off by, the row is chosen again in 64 bits
// (about 1 row in 100 with a sigmoid and a bias).
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
    // A score is off by less than 2^-18 (two units of the fast exp, its
    // rounded exponent x with x e^-x, ten levels of the sum, whose terms'
    // exponents average below ln 1024, and the quotient).
    constexpr float kScoreOff = 0x1p-18f;
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
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) key[j] = key_of(c[j], j);
    }
    // Half of what two keys' values may differ by and yet be in the other
    // order: the score's error, a rounding of the sum, a unit of the last kept bit.
    const float key_off = p.bias ? kScoreOff : 0.0f;
    constexpr float kKeyStep = 0x1p-23f * (N + 1);
    bool sure = true;
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
            const float o = shfl_idx(mine, g), size = shfl_idx(size_of, g);
            ahead += o > mine || (o == mine && g < lane);
            if (lane < p.groups && g != lane && fabsf(o - mine) <= 4.0f * kScoreOff + kKeyStep * (size + size_of)) sure = false;
        }
        const uint32_t kept = __ballot_sync(kFullMask, lane < p.groups && ahead < p.groups_kept);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t e = lane * N + j;
            if (e < p.experts && !(kept >> (e / p.group_size) & 1u)) key[j] = 0;
        }
    }
    sort_falling<N>(key);  // each lane's; the row's next is the largest head
    if (p.groups > 1 && p.group_lanes) {
        // A group is a power of two of whole lanes, which share the comparisons.
        auto value = [&](uint32_t k) {
            const float v = key_value(k & ~kLow);
            return !k ? -INFINITY : p.bias ? v : score(v);
        };
        float a = value(key[0]), b = N > 1 ? value(key[N > 1]) : -INFINITY;  // best and second
        for (uint32_t d = 1; d < p.group_lanes; d *= 2) {
            const float oa = shfl_xor(a, d), ob = shfl_xor(b, d);
            b = fmaxf(fmaxf(b, ob), fminf(a, oa));
            a = fmaxf(a, oa);
        }
        if (!p.top2 || !(b > -INFINITY)) b = 0.0f;
        const float mine = a + b, size_of = mine > -INFINITY ? fabsf(a) + fabsf(b) : 0.0f;
        // A logit's unit, |l| kKeyStep, is one of its score times |l| at most:
        // |x s'(x)| < 1 for a sigmoid, and |l| <= |max| + (max - l) for a softmax.
        const float step = p.bias ? kKeyStep : kKeyStep * (1.0f + fabsf(m)), least = 4.0f * (kScoreOff + kKeyStep);
        const uint32_t own = lane >> p.group_shift, share = lane & (p.group_lanes - 1);
        uint32_t ahead = 0;
        for (uint32_t g = share; g < p.groups + share; g += p.group_lanes) {
            const uint32_t from = g << p.group_shift;
            const float o = __shfl_sync(kFullMask, mine, from), size = __shfl_sync(kFullMask, size_of, from);
            if (g < p.groups && own < p.groups && g != own) {
                ahead += o > mine || (o == mine && g < own);
                if (fabsf(o - mine) <= least + step * (size + size_of)) sure = false;
            }
        }
        for (uint32_t d = 1; d < p.group_lanes; d *= 2) ahead += __shfl_xor_sync(kFullMask, ahead, d);
        if (ahead >= p.groups_kept) {
#pragma unroll
            for (int j = 0; j < N; ++j) key[j] = 0;
        }
    }
    __shared__ uint2 winners[kRouteWarps][32];
    uint2 *won_by = winners[threadIdx.x >> 5];
    const uint32_t turns = min(p.k + 1, 32u), lower = (1u << lane) - 1;
    won_by[lane] = make_uint2(0, 0);
    __syncwarp();
    for (uint32_t i = 0; i < turns; ++i) {
        const uint32_t head = key[0] & ~kLow;
        const uint32_t best = __reduce_max_sync(kFullMask, head);
        const uint32_t owners = __ballot_sync(kFullMask, head == best);
        if (head == best && !(owners & lower)) {  // the lowest of them
            won_by[i] = make_uint2(key[0], lane * N);
#pragma unroll
            for (int j = 0; j + 1 < N; ++j) key[j] = key[j + 1];
            key[N - 1] = 0;
        }
    }
    __syncwarp();
    const uint2 won = won_by[lane];  // key 0: none is left
    // Equal keys of the logits themselves (16-bit types lose nothing in the
    // low bits) are equal logits, which the lanes' order has settled.
    const bool exact = !p.bias && sizeof(T) == 2;
    if (!exact && lane < p.k && won.x) {
        const uint32_t next = lane < 31 ? won_by[lane + 1].x : 0;
        const float a = key_value(won.x & ~kLow), b = key_value(next & ~kLow);
        if (next && a - b <= 2.0f * (key_off + fabsf(a) * kKeyStep) + 0x1p-120f) sure = false;
    }
    int32_t pick = won.x && lane < p.k ? (int32_t)(won.y + kLow - (won.x & kLow)) : -1;
    if (p.k == 32 && !exact) sure = false;  // there is no lane for the 33rd
    if (!__all_sync(kFullMask, sure)) pick = choose_exactly<T, N>(p, src);
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
template <typename T, int N> __global__ void __launch_bounds__(32 * kRouteWarps) route_grad_kernel(const __grid_constant__ RouteGradParams p) {
    const uint32_t lane = threadIdx.x & 31, row = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    const T *src = static_cast<const T *>(p.logits) + row * p.stride;
    const bool whole = !p.sigmoid && !p.renormalize;  // every logit has a gradient
    float l[N], m = -INFINITY, z = 0.0f;
    if (whole) {
        load_run<T, N>(src, lane * N, p.experts, l);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (!(l[j] == l[j])) l[j] = -INFINITY;
            m = fmaxf(m, l[j]);
        }
        m = warp_max(m);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            l[j] = l[j] > -INFINITY ? exp_below(l[j], m) : 0.0f;
            z += l[j];
        }
        z = warp_sum(z);
    }
    uint32_t pick = ~0u;
    float logit = 0.0f, g = 0.0f;
    if (lane < p.k) {
        pick = (uint32_t)p.picks[row * p.picks_stride + lane];
        if (pick < p.experts) {
            g = p.dweights[row * p.dweights_stride + lane];
            logit = to_f32(src[pick]);
        }
    }
    const bool chosen = pick < p.experts && logit > -INFINITY;
    if (!chosen) g = 0.0f;
    const float r = choice_weight(logit, chosen, p.sigmoid, p.renormalize, m, z);
    const float dot = warp_sum(g * r);
    float d = p.scale * r * (p.renormalize ? g - dot : g);
    if (p.sigmoid) d /= 1.0f + expf(logit);
    float dl[N];
#pragma unroll
    for (int j = 0; j < N; ++j) dl[j] = whole && z > 0.0f ? -p.scale * dot * (l[j] / z) : 0.0f;
    // Choices in turn, so that an expert named twice gets both in order.
    for (uint32_t i = 0; i < p.k; ++i) {
        const uint32_t e = __shfl_sync(kFullMask, pick, i);
        const float add = __shfl_sync(kFullMask, d, i);
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (e == lane * N + j) dl[j] += add;
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
