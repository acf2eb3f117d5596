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

// One cluster sorts everything.  Block c takes the c-th part of the places,
// warp w of it the w-th part of those, 32 adjacent places a step, so counts
// and ranks follow the places' order and no result hangs on the order of
// atomics (there are none).
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

    for (uint32_t i = t; i < kOrderWarps * experts; i += kOrderThreads) hist[i] = 0;
    __syncthreads();
    for (uint64_t at = begin; at < end; at += 32) {
        const uint32_t e = at + lane < end ? (uint32_t)picks[at + lane] : ~0u;
        const uint32_t peers = __match_any_sync(kFullMask, e);
        if (e < experts && (peers & ((1u << lane) - 1)) == 0) mine[e] += __popc(peers);
        __syncwarp();
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
    for (uint64_t at = begin; at < end; at += 32) {
        const bool in = at + lane < end;
        const uint32_t e = in ? (uint32_t)picks[at + lane] : ~0u;
        const uint32_t peers = __match_any_sync(kFullMask, e);
        const uint32_t lower = peers & ((1u << lane) - 1);
        const bool taken_up = e < experts;
        const uint32_t place = taken_up ? mine[e] + __popc(lower) : 0;
        __syncwarp();
        if (taken_up) {
            if (lower == 0) mine[e] += __popc(peers);
            order[place] = (int32_t)(at + lane);
        }
        if (in) slot[at + lane] = taken_up ? (int32_t)place : -1;
        __syncwarp();
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
