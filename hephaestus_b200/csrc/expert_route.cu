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
    const float top = warp_max(chosen ? l : -INFINITY);
    float s = 0.0f;
    if (chosen) s = sigmoid ? expf(fminf(l, 0.0f) - fminf(top, 0.0f)) / (1.0f + expf(-fabsf(l))) : exp_below(l, top);
    const float sum = warp_sum(s);
    return sum > 0.0f ? s / sum : 0.0f;
}

// A warp per row; lane i holds experts i, i + 32, ...  What is chosen is
// decided in 64 bits, where two experts' sums with the bias may be near.
template <typename T, int N> __global__ void __launch_bounds__(32 * kRouteWarps) route_kernel(RouteParams p) {
    const uint32_t lane = threadIdx.x & 31, row = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    const T *src = static_cast<const T *>(p.logits) + row * p.stride;
    float l[N], m = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t e = lane + 32 * j;
        l[j] = e < p.experts ? to_f32(src[e]) : -INFINITY;
        if (!(l[j] == l[j])) l[j] = -INFINITY;
        m = fmaxf(m, l[j]);
    }
    m = warp_max(m);
    float z = 0.0f;
    if (!p.sigmoid && !p.renormalize) {
#pragma unroll
        for (int j = 0; j < N; ++j) z += l[j] > -INFINITY ? exp_below(l[j], m) : 0.0f;
        z = warp_sum(z);
    }
    // open: experts that may still be chosen, a bit per j.
    uint32_t open = 0;
    double c[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        open |= (l[j] > -INFINITY ? 1u : 0u) << j;
        c[j] = l[j];
    }
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
                const uint32_t e = lane + 32 * j;
                if (e < p.experts) c[j] += p.bias[e];
                if (!(c[j] > -INFINITY)) open &= ~(1u << j);
            }
        }
        if (p.groups > 1) {
            const uint32_t size = p.experts / p.groups;
            double mine = -INFINITY;  // lane g: the value of group g
            for (uint32_t g = 0; g < p.groups; ++g) {
                double a = -INFINITY, b = -INFINITY;  // best and second
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const uint32_t e = lane + 32 * j;
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
                const uint32_t e = lane + 32 * j;
                if (e < p.experts && !(kept >> (e / size) & 1u)) open &= ~(1u << j);
            }
            if (!p.bias) {
#pragma unroll
                for (int j = 0; j < N; ++j) c[j] = l[j];
            }
        }
    }
    int32_t pick = -1;
    float logit = 0.0f;
    for (uint32_t i = 0; i < p.k; ++i) {
        double best = -INFINITY;
        uint32_t at = 0xffffffffu;
        float of = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if ((open >> j & 1u) && (at == 0xffffffffu || c[j] > best)) {
                best = c[j];
                at = lane + 32 * j;
                of = l[j];
            }
        }
        const uint32_t own = at;
        warp_arg_fold<double, OP_MAX>(best, at);
        if (at == 0xffffffffu) break;  // nothing left, for every lane
        const uint32_t from = at & 31;
        of = __shfl_sync(kFullMask, of, from);
        if (lane == from) open &= ~(1u << (own >> 5));
        if (lane == i) {
            pick = (int32_t)at;
            logit = of;
        }
    }
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
template <typename T, int N> __global__ void __launch_bounds__(32 * kRouteWarps) route_grad_kernel(RouteGradParams p) {
    const uint32_t lane = threadIdx.x & 31, row = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    const T *src = static_cast<const T *>(p.logits) + row * p.stride;
    const bool whole = !p.sigmoid && !p.renormalize;  // every logit has a gradient
    float l[N], m = -INFINITY, z = 0.0f;
    if (whole) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t e = lane + 32 * j;
            l[j] = e < p.experts ? to_f32(src[e]) : -INFINITY;
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
            if (e == lane + 32 * j) dl[j] += add;
    }
    T *out = static_cast<T *>(p.dlogits) + (int64_t)row * p.experts;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t e = lane + 32 * j;
        if (e < p.experts) out[e] = from_f32<T>(dl[j]);
    }
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
    const RouteParams p{a.logits.ptr, a.bias, a.logits.stride, a.rows, a.experts, a.k, a.groups, a.groups_kept,
                        a.sigmoid, a.renormalize, a.group_top == 2, a.scale, a.weights, a.picks};
    const dim3 grid((a.rows + kRouteWarps - 1) / kRouteWarps);
    return dispatch_row_dtype(a.dtype, [&]<typename T>() {
        return dispatch_experts(a.experts, [&]<int N>() {
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
