// expert_order.cu — the order of routed (token, choice) pairs by expert: a
// stable counting sort with its exclusive offsets and its inverse.
//
//   offsets[e] = number of pairs of experts below e
//   order      = the pairs' places, by expert and then by place
//   slot       = the inverse of order (-1 for a pair that no expert takes)
//
// Places are dealt in equal runs to blocks, of these to warps, and of these 32
// adjacent ones to a step, so that counts of "all before" follow the places'
// order.  Bytes: 12 a pair; bound by the latency of three dependent phases
// (counts, their prefixes, places), and past 65536 pairs also by the counts of
// all blocks, which every block of the second launch reads: 512 x 512 x experts
// words at the most (131072 x 8 pairs of 256 / 1024 experts: 46 / 97 us).
#include <cooperative_groups.h>

#include "row_ops.h"
#include "row_utils.cuh"

namespace heph {

namespace {

namespace cg = cooperative_groups;

constexpr int kFew = 256, kMany = 1024;  // threads of a block that works alone, and of others
constexpr int kSteps = 4;                // steps of a warp whose picks are loaded together
constexpr uint32_t kMaxBlocks = 512;     // blocks whose counts are read by every block

// The lanes whose pick is this lane's, from a vote on each bit of the picks.
// (match.any takes a turn for each different value: 2.3 times the kernel's
// time at 262144 pairs of 256 experts.)
__device__ __forceinline__ uint32_t lanes_alike(uint32_t e, bool has, int bits) {
    uint32_t peers = __ballot_sync(kFullMask, has);
    for (int b = 0; b < bits; ++b) {
        const uint32_t ones = __ballot_sync(kFullMask, e >> b & 1u);
        peers &= e >> b & 1u ? ones : ~ones;
    }
    return peers;
}

// A block's part of the places, its warps' counts per expert, and the walks
// over both.
template <int THREADS> struct OrderPart {
    static constexpr int kWarps = THREADS / 32;
    static constexpr uint32_t kExpertsPerThread = kMaxExperts / THREADS;
    const int32_t *picks;
    uint32_t experts, bits, lane;
    uint64_t begin, end;   // places of this warp
    uint32_t *hist, *mine;  // [kWarps][experts], of this warp
    uint32_t first[kSteps];

    __device__ OrderPart(const int32_t *picks_, uint32_t count, uint32_t experts_, uint32_t blocks, uint32_t block, uint32_t *hist_)
        : picks(picks_), experts(experts_), hist(hist_) {
        const uint32_t warp = threadIdx.x >> 5;
        bits = 32 - __clz(experts - 1);
        lane = threadIdx.x & 31;
        // Places per warp: a multiple of 32, so that only the last step is ragged.
        const uint64_t per_warp = ((uint64_t)count + blocks * THREADS - 1) / (blocks * THREADS) * 32;
        begin = per_warp * (block * kWarps + warp);
        end = min(begin + per_warp, (uint64_t)count);
        mine = hist + warp * experts;
        load(begin, first);
        for (uint32_t i = threadIdx.x; i < kWarps * experts; i += THREADS) hist[i] = 0;
        __syncthreads();
    }
    __device__ __forceinline__ void load(uint64_t at, uint32_t (&e)[kSteps]) const {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) e[i] = at + 32 * i + lane < end ? (uint32_t)picks[at + 32 * i + lane] : ~0u;
    }
    // f(place of the step, this lane's pick) for every step of 32 places; the
    // first batch (mostly the only one) is in registers already.
    template <typename F> __device__ __forceinline__ void each_step(F &&f) const {
        for (uint64_t at = begin; at < end; at += 32 * kSteps) {
            uint32_t e[kSteps];
            if (at == begin) {
#pragma unroll
                for (int i = 0; i < kSteps; ++i) e[i] = first[i];
            } else {
                load(at, e);
            }
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                if (at + 32 * i >= end) break;
                f(at + 32 * i, e[i]);
            }
        }
    }
    // Counts; then hist is the counts of the warps below, and the block's of
    // expert t, t + THREADS, ... are returned.
    __device__ __forceinline__ void count(uint32_t (&total)[kExpertsPerThread]) const {
        each_step([&](uint64_t, uint32_t e) {
            if (e < experts) atomicAdd(&mine[e], 1u);  // a count does not depend on the order
        });
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kExpertsPerThread; ++i) {
            const uint32_t e = threadIdx.x + i * THREADS;
            total[i] = 0;
            if (e >= experts) continue;
            uint32_t n[kWarps];
#pragma unroll
            for (int w = 0; w < kWarps; ++w) n[w] = hist[w * experts + e];
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                hist[w * experts + e] = total[i];
                total[i] += n[w];
            }
        }
    }
    // Places by expert, given each expert's count in the blocks below and in
    // all; returns how many pairs are taken.
    __device__ __forceinline__ uint32_t place(const uint32_t (&before)[kExpertsPerThread], const uint32_t (&all)[kExpertsPerThread],
                                              bool first_block, int32_t *offsets, int32_t *order, int32_t *slot) const {
        __shared__ uint32_t warp_total[kWarps];
        const uint32_t t = threadIdx.x, warp = t >> 5;
        uint32_t taken = 0;  // exclusive prefix of the counts over the experts, THREADS at a time
        for (uint32_t i = 0; i < kExpertsPerThread && i * THREADS < experts; ++i) {
            uint32_t upto = all[i];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t o = __shfl_up_sync(kFullMask, upto, d);
                if (lane >= d) upto += o;
            }
            __syncthreads();
            if (lane == 31) warp_total[warp] = upto;
            __syncthreads();
            uint32_t start = taken + upto - all[i];
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                start += w < warp ? warp_total[w] : 0;
                taken += warp_total[w];
            }
            const uint32_t e = t + i * THREADS;
            if (e < experts) {
#pragma unroll
                for (int w = 0; w < kWarps; ++w) hist[w * experts + e] += start + before[i];
                if (first_block) offsets[e] = (int32_t)start;
            }
        }
        if (first_block && t == 0) offsets[experts] = (int32_t)taken;
        __syncthreads();
        each_step([&](uint64_t at, uint32_t e) {
            const bool has = e < experts;
            const uint32_t peers = lanes_alike(e, has, bits), lower = peers & ((1u << lane) - 1);
            const uint32_t to = has ? mine[e] + __popc(lower) : 0;
            __syncwarp();
            if (has) {
                if (lower == 0) mine[e] += __popc(peers);
                order[to] = (int32_t)(at + lane);
            }
            if (at + lane < end) slot[at + lane] = has ? (int32_t)to : -1;
            __syncwarp();
        });
        return taken;
    }
};

__device__ __forceinline__ void fill_rest(int32_t *order, uint64_t from, uint32_t count, uint32_t blocks, uint32_t block) {
    for (uint64_t i = from + (uint64_t)block * blockDim.x + threadIdx.x; i < count; i += blocks * blockDim.x) order[i] = -1;
}

// One block, or a cluster whose blocks read each other's counts.
template <int THREADS> __global__ void __launch_bounds__(THREADS) expert_order_kernel(const int32_t *picks, uint32_t count, uint32_t experts,
                                                                     int32_t *offsets, int32_t *order, int32_t *slot) {
    extern __shared__ uint32_t smem[];
    using Part = OrderPart<THREADS>;
    uint32_t *counts = smem + Part::kWarps * experts;  // [experts]: this block's, read by the cluster
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t blocks = cluster.num_blocks(), block = cluster.block_rank();
    const Part part(picks, count, experts, blocks, block, smem);
    uint32_t before[Part::kExpertsPerThread] = {}, all[Part::kExpertsPerThread];
    part.count(all);
    if (blocks > 1) {
#pragma unroll
        for (uint32_t i = 0; i < Part::kExpertsPerThread; ++i)
            if (threadIdx.x + i * THREADS < experts) counts[threadIdx.x + i * THREADS] = all[i];
        cluster.sync();
#pragma unroll
        for (uint32_t i = 0; i < Part::kExpertsPerThread; ++i) {
            const uint32_t e = threadIdx.x + i * THREADS;
            if (e >= experts) continue;
            all[i] = 0;
#pragma unroll
            for (uint32_t b = 0; b < 16; ++b) {
                const uint32_t n = b < blocks ? cluster.map_shared_rank(counts, b)[e] : 0;
                before[i] += b < block ? n : 0;
                all[i] += n;
            }
        }
    }
    const uint32_t taken = part.place(before, all, block == 0, offsets, order, slot);
    fill_rest(order, taken, count, blocks, block);
    if (blocks > 1) cluster.sync();  // no block leaves while its counts may be read
}

// More places than one cluster takes: each block's counts go to `counts`
// [blocks][pitch], and every block of the next launch reads them all, four
// experts a load and the rows shared out among its threads.
__host__ __device__ constexpr uint32_t counts_pitch(uint32_t experts) { return (experts + 3) / 4 * 4; }
__global__ void __launch_bounds__(kMany) expert_count_kernel(const int32_t *picks, uint32_t count, uint32_t experts, uint32_t *counts) {
    extern __shared__ uint32_t smem[];
    let_next_start();
    using Part = OrderPart<kMany>;
    const Part part(picks, count, experts, gridDim.x, blockIdx.x, smem);
    uint32_t total[Part::kExpertsPerThread];
    part.count(total);
#pragma unroll
    for (uint32_t i = 0; i < Part::kExpertsPerThread; ++i) {
        const uint32_t e = threadIdx.x + i * kMany;
        if (e < experts) counts[blockIdx.x * counts_pitch(experts) + e] = total[i];
    }
}
__global__ void __launch_bounds__(kMany) expert_place_kernel(const int32_t *picks, uint32_t count, uint32_t experts, const uint32_t *counts,
                                                                     int32_t *offsets, int32_t *order, int32_t *slot) {
    extern __shared__ uint32_t smem[];
    __shared__ uint32_t sums[2][kMaxExperts];  // of the blocks below, of all
    for (uint32_t e = threadIdx.x; e < kMaxExperts; e += kMany) sums[0][e] = sums[1][e] = 0;
    using Part = OrderPart<kMany>;
    const Part part(picks, count, experts, gridDim.x, blockIdx.x, smem);
    uint32_t before[Part::kExpertsPerThread] = {}, all[Part::kExpertsPerThread];
    part.count(all);
    after_previous();  // its own counts need nothing of the first launch
    const uint32_t pitch = counts_pitch(experts), quads = pitch / 4, rows = kMany / quads;
    const uint32_t quad = threadIdx.x % quads, first = threadIdx.x / quads;
    if (first < rows) {
        uint32_t low[4] = {}, sum[4] = {};
#pragma unroll 8
        for (uint32_t b = first; b < gridDim.x; b += rows) {
            const auto n = *reinterpret_cast<const Pack<uint32_t, 4> *>(counts + b * pitch + quad * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                low[j] += b < blockIdx.x ? n.e[j] : 0;
                sum[j] += n.e[j];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (quad * 4 + j >= experts) continue;  // past the last: not written
            atomicAdd(&sums[0][quad * 4 + j], low[j]);
            atomicAdd(&sums[1][quad * 4 + j], sum[j]);
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < Part::kExpertsPerThread; ++i) {
        const uint32_t e = threadIdx.x + i * kMany;
        before[i] = e < experts ? sums[0][e] : 0;
        all[i] = e < experts ? sums[1][e] : 0;
    }
    const uint32_t taken = part.place(before, all, blockIdx.x == 0, offsets, order, slot);
    fill_rest(order, taken, count, gridDim.x, blockIdx.x);
}

// Two steps for each warp of 2048 places, while the blocks are few enough.
uint32_t blocks_of(uint32_t count) { return std::min(kMaxBlocks, (count + 2 * kMany - 1) / (2 * kMany)); }
// One cluster of up to 16 blocks takes four steps for each warp.
bool one_cluster(uint32_t count) { return count <= 16 * kSteps * kMany; }

size_t order_smem(int threads, uint32_t experts) { return (threads / 32 + 1) * experts * sizeof(uint32_t); }

template <typename K> heph_status allow_smem(K kernel) {
    // The same limit on every call: calls of several threads do not lower it for one another.
    HEPH_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)order_smem(kMany, kMaxExperts)),
                  HEPH_DISPATCH_FAILED, "expert order shared memory");
    return HEPH_OK;
}

}  // namespace

size_t expert_order_workspace(uint32_t count, uint32_t experts) {
    return one_cluster(count) ? 0 : (size_t)blocks_of(count) * counts_pitch(experts) * sizeof(uint32_t);
}

heph_status launch_expert_order(const int32_t *picks, uint32_t count, uint32_t experts, int32_t *offsets,
                                int32_t *order, int32_t *slot, uint32_t *workspace, cudaStream_t stream) {
    // Measured for 64 x 8 / 32768 x 8 pairs of 256 experts: 5.4 / 16.4 us with
    // blocks of 256 threads throughout, 5.8 / 14.3 us with these, and 11.6 with
    // the second launch's own counts during the first.
    if (count <= 2 * kSteps * kFew)
        return launch_clusters("expert order", expert_order_kernel<kFew>, dim3(1), dim3(kFew), 1, order_smem(kFew, experts), stream,
                               picks, count, experts, offsets, order, slot);
    const size_t smem = order_smem(kMany, experts);
    heph_status st;
    if (one_cluster(count)) {
        uint32_t blocks = 1;
        while (blocks < 16 && blocks * kSteps * kMany < count) blocks *= 2;
        st = allow_smem(expert_order_kernel<kMany>);
        if (st != HEPH_OK) return st;
        if (blocks > 8)
            HEPH_CUDA_TRY(cudaFuncSetAttribute(expert_order_kernel<kMany>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1),
                          HEPH_DISPATCH_FAILED, "expert order cluster size");
        return launch_clusters("expert order", expert_order_kernel<kMany>, dim3(blocks), dim3(kMany), blocks, smem, stream,
                               picks, count, experts, offsets, order, slot);
    }
    const dim3 grid(blocks_of(count));
    if ((st = allow_smem(expert_count_kernel)) != HEPH_OK || (st = allow_smem(expert_place_kernel)) != HEPH_OK) return st;
    st = launch_rows("expert counts", expert_count_kernel, grid, dim3(kMany), smem, stream, picks, count, experts, workspace);
    if (st != HEPH_OK) return st;
    return launch_next("expert order", expert_place_kernel, grid, dim3(kMany), smem, stream, picks, count, experts, workspace,
                       offsets, order, slot);
}

}  // namespace heph
