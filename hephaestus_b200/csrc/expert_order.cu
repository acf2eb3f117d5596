// expert_order.cu — the order of routed (token, choice) pairs by expert: a
// stable counting sort with its exclusive offsets and its inverse.
//
//   offsets[e] = number of pairs of experts below e
//   order      = the pairs' places, by expert and then by place
//   slot       = the inverse of order (-1 for a pair that no expert takes)
#include <cooperative_groups.h>

#include "row_ops.h"
#include "row_utils.cuh"

namespace heph {

namespace {

namespace cg = cooperative_groups;

constexpr int kOrderThreads = 1024;
constexpr int kOrderWarps = kOrderThreads / 32;

constexpr int kSteps = 16;  // steps of a warp whose picks are loaded together

__device__ __forceinline__ void load_picks(const int32_t *picks, uint64_t at, uint64_t end, uint32_t (&e)[kSteps]) {
    at += threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) e[i] = at + 32 * i < end ? (uint32_t)picks[at + 32 * i] : ~0u;
}

// The lanes whose pick is this lane's, from a vote on each bit of the picks.
// (match.any takes a turn for each different value: 41 us instead of 9 for
// 262144 pairs of 256 experts.)
__device__ __forceinline__ uint32_t lanes_alike(uint32_t e, bool has, int bits) {
    uint32_t peers = __ballot_sync(kFullMask, has);
    for (int b = 0; b < bits; ++b) {
        const uint32_t ones = __ballot_sync(kFullMask, e >> b & 1u);
        peers &= e >> b & 1u ? ones : ~ones;
    }
    return peers;
}

// One cluster sorts everything.  Block c takes the c-th part of the places,
// warp w of it the w-th part of those, 32 adjacent places a step, so counts
// and ranks follow the places' order.
__global__ void __launch_bounds__(kOrderThreads) expert_order_kernel(const int32_t *picks, uint32_t count, uint32_t experts,
                                                                     int32_t *offsets, int32_t *order, int32_t *slot) {
    extern __shared__ uint32_t smem[];
    uint32_t *hist = smem;                            // [kOrderWarps][experts]
    uint32_t *total = smem + kOrderWarps * experts;   // [experts]: this block's counts, read by the cluster
    __shared__ uint32_t warp_total[kOrderWarps];
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t blocks = cluster.num_blocks(), block = cluster.block_rank();
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
    // Places per warp: a multiple of 32, so only the last step is ragged.
    const uint64_t per_warp = ((uint64_t)count + blocks * kOrderThreads - 1) / (blocks * kOrderThreads) * 32;
    const uint64_t begin = per_warp * (block * kOrderWarps + warp);
    const uint64_t end = begin + per_warp < count ? begin + per_warp : count;
    uint32_t *mine = hist + warp * experts;
    const int bits = 32 - __clz(experts - 1);

    for (uint32_t i = t; i < kOrderWarps * experts; i += kOrderThreads) hist[i] = 0;
    __syncthreads();
    // The picks of kSteps steps are loaded together; the first batch (mostly
    // the only one) stays in registers for the second walk.
    uint32_t first[kSteps];
    load_picks(picks, begin, end, first);
    for (uint64_t at = begin; at < end; at += 32 * kSteps) {
        uint32_t e[kSteps];
        if (at == begin) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) e[i] = first[i];
        } else {
            load_picks(picks, at, end, e);
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            if (at + 32 * i >= end) break;
            if (e[i] < experts) atomicAdd(&mine[e[i]], 1u);  // a count does not depend on the order
        }
    }
    __syncthreads();
    // Counts of the warps below, per expert.
    uint32_t below = 0;
    if (t < experts) {
        for (uint32_t w = 0; w < kOrderWarps; ++w) {
            const uint32_t n = hist[w * experts + t];
            hist[w * experts + t] = below;
            below += n;
        }
        total[t] = below;
    }
    cluster.sync();
    uint32_t before = 0, all = 0;  // counts of the blocks below, and of all
    if (t < experts) {
        for (uint32_t b = 0; b < blocks; ++b) {
            const uint32_t n = cluster.map_shared_rank(total, b)[t];
            before += b < block ? n : 0;
            all += n;
        }
    }
    // Exclusive prefix of the counts over the experts (at most one a thread).
    uint32_t upto = all;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t o = __shfl_up_sync(kFullMask, upto, d);
        if (lane >= d) upto += o;
    }
    if (lane == 31) warp_total[warp] = upto;
    __syncthreads();
    uint32_t start = upto - all, taken = 0;
    for (uint32_t w = 0; w < kOrderWarps; ++w) {
        start += w < warp ? warp_total[w] : 0;
        taken += warp_total[w];
    }
    if (t < experts) {
        for (uint32_t w = 0; w < kOrderWarps; ++w) hist[w * experts + t] += start + before;
        if (block == 0) offsets[t] = (int32_t)start;
    }
    if (block == 0 && t == 0) offsets[experts] = (int32_t)taken;
    __syncthreads();
    for (uint64_t at = begin; at < end; at += 32 * kSteps) {
        uint32_t e[kSteps];
        if (at == begin) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) e[i] = first[i];
        } else {
            load_picks(picks, at, end, e);
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const uint64_t place = at + 32 * i + lane;
            if (at + 32 * i >= end) break;
            const bool has = e[i] < experts;
            const uint32_t peers = lanes_alike(e[i], has, bits);
            const uint32_t lower = peers & ((1u << lane) - 1);
            const uint32_t to = has ? mine[e[i]] + __popc(lower) : 0;
            __syncwarp();
            if (has) {
                if (lower == 0) mine[e[i]] += __popc(peers);
                order[to] = (int32_t)place;
            }
            if (place < end) slot[place] = has ? (int32_t)to : -1;
            __syncwarp();
        }
    }
    for (uint64_t i = taken + (uint64_t)block * kOrderThreads + t; i < count; i += blocks * kOrderThreads) order[i] = -1;
    cluster.sync();  // no block leaves while its counts may be read
}

}  // namespace

heph_status launch_expert_order(const int32_t *picks, uint32_t count, uint32_t experts, int32_t *offsets,
                                int32_t *order, int32_t *slot, cudaStream_t stream) {
    // 4096 places a block, up to the largest cluster.
    uint32_t blocks = 1;
    while (blocks < 16 && (uint64_t)blocks * 4096 < count) blocks *= 2;
    const size_t smem = (kOrderWarps + 1) * experts * sizeof(uint32_t);
    // The same limit on every call: calls of several threads do not lower it for one another.
    HEPH_CUDA_TRY(cudaFuncSetAttribute(expert_order_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (kOrderWarps + 1) * kMaxExperts * sizeof(uint32_t)),
                  HEPH_DISPATCH_FAILED, "expert order shared memory");
    HEPH_CUDA_TRY(cudaFuncSetAttribute(expert_order_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1),
                  HEPH_DISPATCH_FAILED, "expert order cluster size");
    return launch_clusters("expert order", expert_order_kernel, dim3(blocks), dim3(kOrderThreads), blocks, smem, stream,
                           picks, count, experts, offsets, order, slot);
}

}  // namespace heph
