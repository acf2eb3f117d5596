// sample.cu — tokens drawn from rows of logits with temperature, top-k, top-p
// and min-p, from given uniform numbers.
//
//   w_i = exp((l_i - max) / T).  In the order of falling l (equal ones by
//   index): top-k keeps the first k; top-p of those the ones before which less
//   than p of their mass lies; min-p of those the ones of w >= min_p; the first
//   always stays.  The token is the first index whose running sum of kept w
//   exceeds u times the whole.
//
// What is kept is a threshold: all keys above one key and, by index, some of
// those equal to it.  The threshold is found by histograms of keys (counts
// for top-k, masses for top-p) of ever narrower ranges, with no sort.
//
// Masses are whole numbers, w in units of 2^-scale_bits (45 for a vocabulary
// of 2^17), so that sums do not depend on their order: the answer is the same
// in any batch and for any number of blocks per row.
#include <cooperative_groups.h>

#include "row_ops.h"
#include "row_utils.cuh"

namespace heph {

namespace {

namespace cg = cooperative_groups;

constexpr int kSampleThreads = 1024;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kBinBits = 12;
constexpr int kBins = 1 << kBinBits;
constexpr int kBinsPerThread = kBins / kSampleThreads;
constexpr int kMaxCluster = 8;

struct SampleParams {
    const void *logits;
    int64_t stride;
    const float *uniform, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    double temperature_all, top_p_all, min_p_all;
    int32_t top_k_all;
    uint32_t vocab;
    int scale_bits;
    int64_t *tokens;
    float *probs;
};

struct Histogram {
    uint32_t low[kBins], high[kBins];  // 64-bit masses, or counts in `low`
};

struct SampleShared {
    Histogram hist[2];
    float max;
    uint64_t mass;                    // this block's kept mass above the threshold
    uint32_t ties;                    // and its number of keys equal to it
    uint64_t warp_mass[kSampleWarps];
    uint32_t warp_ties[kSampleWarps];
    uint64_t scan[kSampleWarps];
    uint32_t found_bin;
    uint64_t found_above;
};

// Adds a 64-bit mass by two 32-bit atomics, whose order changes nothing.
__device__ __forceinline__ void add_mass(Histogram &h, uint32_t bin, uint64_t mass) {
    const uint32_t low = (uint32_t)mass;
    const uint32_t old = atomicAdd(&h.low[bin], low);
    const uint32_t high = (uint32_t)(mass >> 32) + (old + low < old);
    if (high) atomicAdd(&h.high[bin], high);
}

__device__ __forceinline__ uint64_t warp_scan(uint64_t v) {  // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t o = shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// One row, seen by one block of its cluster: the block takes an equal part of
// the row's 16-byte vectors, each of its warps an equal part of those, so
// that blocks, warps, steps, lanes and elements are in the order of indices.
template <typename T> struct RowPart {
    static constexpr int V = 16 / sizeof(T);
    const T *row;
    uint32_t vocab, lead;  // lead: elements of the first vector before the row
    uint32_t begin, end;   // vectors of this warp

    __device__ RowPart(const T *row_, uint32_t vocab_, uint32_t parts, uint32_t part) : row(row_), vocab(vocab_) {
        lead = (uint32_t)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
        const uint32_t vectors = (lead + vocab + V - 1) / V;
        const uint32_t each = ((vectors + parts - 1) / parts + 31) / 32 * 32;
        begin = min(each * part, vectors);
        end = min(begin + each, vectors);
    }
    // Elements of vector q; those outside the row are NaN.
    __device__ __forceinline__ void load(uint32_t q, float (&v)[V]) const {
        const int64_t at = (int64_t)q * V - lead;
        if (at >= 0 && at + V <= vocab) {
            const auto u = *reinterpret_cast<const Pack<T, V> *>(row + at);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = to_f32(u.e[j]);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = at + j >= 0 && at + j < vocab ? to_f32(row[at + j]) : NAN;
        }
    }
    // f(logit) for every element of the warp's part.
    template <typename F> __device__ __forceinline__ void each(F &&f) const {
        for (uint32_t q = begin + (threadIdx.x & 31); q < end; q += 32) {
            float v[V];
            load(q, v);
#pragma unroll
            for (int j = 0; j < V; ++j) f(v[j]);
        }
    }
};

struct Weigher {
    float max;
    double inverse_t, unit, least;  // unit = 2^scale_bits; least: min_p
    __device__ __forceinline__ double weight(float l) const {
        return l == max ? 1.0 : exp(((double)l - (double)max) * inverse_t);
    }
    __device__ __forceinline__ uint64_t mass(float l) const { return __double2ull_rn(weight(l) * unit); }
    // The mass, or none where min-p drops it.
    __device__ __forceinline__ uint64_t kept_mass(float l) const {
        const double w = weight(l);
        return w >= least ? __double2ull_rn(w * unit) : 0;
    }
};

// Everything that is kept: keys above `key`, and the first `ties` equal to it.
struct Threshold {
    uint32_t key, ties;
};

struct Narrowed {
    uint32_t key;
    uint64_t above;  // count or mass of the keys above `key`
    uint64_t wanted;
};

// The largest key whose keys-at-or-above hold at least wanted = need(total)
// (counts, or with MASS masses), among the row's keys above `floor`, of which
// `total` is the whole; key = floor where these do not reach it.  First by 4096 equal steps of the logit below the
// maximum (a window of `window`; the last bin takes the rest), which spreads
// any scale of logits; then, within one bin, by steps of the key.
template <bool MASS, typename T, typename Need>
__device__ Narrowed narrow(const RowPart<T> &part, const Weigher &weigh, SampleShared &s, int &turn, uint32_t floor,
                           float window, Need &&need) {
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const float max = weigh.max, steps = kBins / window;
    auto linear_bin = [&](float l) -> uint32_t {
        return l == max ? 0 : (uint32_t)fminf((max - l) * steps, (float)(kBins - 1));
    };
    Narrowed got{floor, 0, 0};
    uint32_t first = 0, high = ordered_key(max), low = floor + 1;
    int shift = -1;  // -1: the linear bins
    for (;;) {
        Histogram &h = s.hist[turn];
        turn ^= 1;
        for (int i = t; i < kBins; i += kSampleThreads) h.low[i] = h.high[i] = 0;
        __syncthreads();
        part.each([&](float l) {
            if (!(l == l)) return;
            const uint32_t key = ordered_key(l);
            if (key < low || key > high) return;
            uint32_t bin = linear_bin(l);
            if (shift >= 0) {
                if (bin != first) return;
                bin = (high - key) >> shift;
            }
            if constexpr (MASS) {
                const uint64_t mass = weigh.mass(l);
                if (mass) add_mass(h, bin, mass);
            } else {
                atomicAdd(&h.low[bin], 1u);
            }
        });
        cluster.sync();
        // Every block of the cluster sums all their histograms and finds the
        // bin by itself.  The other histogram is cleared after the next
        // barrier at the earliest, when nobody reads this one.
        uint64_t bins[kBinsPerThread], sum = 0;
#pragma unroll
        for (int i = 0; i < kBinsPerThread; ++i) bins[i] = 0;
        for (uint32_t b = 0; b < cluster.num_blocks(); ++b) {
            const Histogram *o = cluster.map_shared_rank(&h, b);
            const Pack<uint32_t, kBinsPerThread> lo = *reinterpret_cast<const Pack<uint32_t, kBinsPerThread> *>(&o->low[t * kBinsPerThread]);
            const Pack<uint32_t, kBinsPerThread> hi = *reinterpret_cast<const Pack<uint32_t, kBinsPerThread> *>(&o->high[t * kBinsPerThread]);
#pragma unroll
            for (int i = 0; i < kBinsPerThread; ++i) bins[i] += (uint64_t)hi.e[i] << 32 | lo.e[i];
        }
#pragma unroll
        for (int i = 0; i < kBinsPerThread; ++i) sum += bins[i];
        uint64_t upto = warp_scan(sum);
        if (lane == 31) s.scan[warp] = upto;
        if (t == 0) s.found_bin = kBins;
        __syncthreads();
        uint64_t below = 0, all = 0;
        for (int w = 0; w < kSampleWarps; ++w) {
            below += w < (int)warp ? s.scan[w] : 0;
            all += s.scan[w];
        }
        if (shift < 0) got.wanted = need(all);
        uint64_t run = got.above + below + upto - sum;
#pragma unroll
        for (int i = 0; i < kBinsPerThread; ++i) {
            if (run < got.wanted && run + bins[i] >= got.wanted) {
                s.found_bin = t * kBinsPerThread + i;
                s.found_above = run;
            }
            run += bins[i];
        }
        __syncthreads();
        const uint32_t bin = s.found_bin;
        if (bin == kBins) {  // these keys do not reach it
            got.above = all;
            return got;
        }
        got.above = s.found_above;
        if (shift < 0) {
            // The keys of linear bin `bin`, with a margin for the rounding of
            // the bin's number; which of them belong is decided by that number.
            first = bin;
            const double width = (double)window / kBins, margin = 1e-6;
            if (bin) high = min(high, ordered_key(__double2float_ru((double)max - bin * width * (1.0 - margin))));
            if (bin < kBins - 1) low = ::max(low, ordered_key(__double2float_rd((double)max - (bin + 1) * width * (1.0 + margin))));
        } else {
            high -= bin << shift;
            low = ::max(low, high - ((1u << shift) - 1));
        }
        if (low == high) {
            got.key = low;
            return got;
        }
        shift = ::max(0, 32 - __clz(high - low) - kBinBits);
    }
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const __grid_constant__ SampleParams p) {
    extern __shared__ __align__(16) unsigned char raw[];
    SampleShared &s = *reinterpret_cast<SampleShared *>(raw);
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t blocks = cluster.num_blocks(), block = cluster.block_rank();
    const uint32_t row = blockIdx.x / blocks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const RowPart<T> part(static_cast<const T *>(p.logits) + row * p.stride, p.vocab, blocks * kSampleWarps,
                          block * kSampleWarps + warp);

    float max = -INFINITY;
    part.each([&](float l) { max = fmaxf(max, l); });  // fmaxf passes NaN over
    max = warp_max(max);
    if (lane == 0) s.warp_mass[warp] = __float_as_uint(max);
    __syncthreads();
    if (warp == 0) {
        max = warp_max(__uint_as_float((uint32_t)s.warp_mass[lane]));
        if (lane == 0) s.max = max;
    }
    cluster.sync();
    max = -INFINITY;
    for (uint32_t b = 0; b < blocks; ++b) max = fmaxf(max, *cluster.map_shared_rank(&s.max, b));
    if (max == -INFINITY) {  // nothing to choose from
        if (block == 0 && threadIdx.x == 0) {
            p.tokens[row] = -1;
            p.probs[row] = 0.0f;
        }
        cluster.sync();
        return;
    }

    const double t = p.temperature ? p.temperature[row] : p.temperature_all;
    const int32_t k = p.top_k ? p.top_k[row] : p.top_k_all;
    const double top_p = p.top_p ? p.top_p[row] : p.top_p_all;
    const double min_p = p.min_p ? p.min_p[row] : p.min_p_all;
    const bool greedy = !(t > 0.0) || k == 1;
    const Weigher weigh{max, greedy ? 1.0 : 1.0 / t, ldexp(1.0, p.scale_bits), min_p > 0.0 ? fmin(min_p, 1.0) : 0.0};

    Threshold keep{0, 0};  // no key is 0: everything
    int turn = 0;
    if (greedy) {
        keep = {ordered_key(max), 1};
    } else {
        if (k > 0 && (uint32_t)k < p.vocab) {
            const Narrowed n = narrow<false>(part, weigh, s, turn, 0, 16.0f, [&](uint64_t) { return (uint64_t)k; });
            if (n.key) keep = {n.key, (uint32_t)(k - n.above)};
        }
        if (top_p < 1.0) {
            const uint64_t tie = keep.ties ? weigh.mass(key_value(keep.key)) : 0;
            const float window = (float)fmin(fmax(32.0 * t, 0x1p-10), 0x1p10);
            const Narrowed n = narrow<true>(part, weigh, s, turn, keep.key, window, [&](uint64_t above) -> uint64_t {
                const uint64_t all = above + keep.ties * tie;
                const double part_of = ceil((double)all * (top_p > 0.0 ? top_p : 0.0));
                return part_of < 1.0 ? 1 : ::min((uint64_t)part_of, all);
            });
            const uint64_t left = n.wanted - n.above;  // > 0, to be filled by keys equal to n.key
            const uint64_t each = n.key == keep.key ? tie : weigh.mass(key_value(n.key));
            keep = {n.key, each ? (uint32_t)((left + each - 1) / each) : keep.ties};
        }
    }

    // Kept mass and ties, per warp, block and row.
    const uint64_t tie = keep.ties ? weigh.kept_mass(key_value(keep.key)) : 0;
    uint64_t mass = 0;
    uint32_t ties = 0;
    part.each([&](float l) {
        if (!(l == l)) return;
        const uint32_t key = ordered_key(l);
        if (key > keep.key) mass += weigh.kept_mass(l);
        ties += key == keep.key;
    });
    mass = warp_fold<int64_t, OP_SUM>((int64_t)mass);
    ties = warp_fold<uint32_t, OP_SUM>(ties);
    if (lane == 0) {
        s.warp_mass[warp] = mass;
        s.warp_ties[warp] = ties;
    }
    __syncthreads();
    if (warp == 0) {
        const uint64_t m = (uint64_t)warp_fold<int64_t, OP_SUM>((int64_t)s.warp_mass[lane]);
        const uint32_t n = warp_fold<uint32_t, OP_SUM>(s.warp_ties[lane]);
        if (lane == 0) {
            s.mass = m;
            s.ties = n;
        }
    }
    cluster.sync();
    auto kept = [&](uint64_t m, uint64_t n) { return m + (n < keep.ties ? n : keep.ties) * tie; };
    uint64_t all_mass = 0, at_mass = 0;
    uint32_t all_ties = 0, at_ties = 0;
    for (uint32_t b = 0; b < blocks; ++b) {
        const uint64_t m = *cluster.map_shared_rank(&s.mass, b);
        const uint32_t n = *cluster.map_shared_rank(&s.ties, b);
        if (b < block) {
            at_mass += m;
            at_ties += n;
        }
        all_mass += m;
        all_ties += n;
    }
    cluster.sync();  // the last reads of other blocks' memory
    const uint64_t all = kept(all_mass, all_ties);
    const float u = p.uniform[row];
    const uint64_t point = ::min((uint64_t)((u > 0.0f ? (double)fminf(u, 1.0f) : 0.0) * (double)all), all - 1);
    // The warp in whose part the running sum passes the point walks its part.
    for (uint32_t w = 0; w < warp; ++w) {
        at_mass += s.warp_mass[w];
        at_ties += s.warp_ties[w];
    }
    if (point < kept(at_mass, at_ties) || point >= kept(at_mass + mass, at_ties + ties)) return;
    for (uint32_t q0 = part.begin; q0 < part.end; q0 += 32) {
        constexpr int V = RowPart<T>::V;
        float v[V];
        uint64_t m[V], sum = 0;
        uint32_t n = 0;
        if (q0 + lane < part.end) part.load(q0 + lane, v);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            m[j] = 0;
            if (q0 + lane >= part.end || !(v[j] == v[j])) v[j] = NAN;
            else if (ordered_key(v[j]) > keep.key) m[j] = weigh.kept_mass(v[j]);
            sum += m[j];
            n += v[j] == v[j] && ordered_key(v[j]) == keep.key;
        }
        uint64_t end_mass = at_mass + warp_scan(sum);
        const uint64_t end_ties = at_ties + warp_scan((uint64_t)n);
        const bool here = point >= kept(end_mass - sum, end_ties - n) && point < kept(end_mass, end_ties);
        if (here) {
            uint64_t run_mass = end_mass - sum;
            uint64_t run_ties = end_ties - n;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (!(v[j] == v[j])) continue;
                const uint64_t before = kept(run_mass, run_ties);
                run_mass += m[j];
                run_ties += ordered_key(v[j]) == keep.key;
                if (point >= before && point < kept(run_mass, run_ties)) {
                    p.tokens[row] = (int64_t)(q0 + lane) * V - part.lead + j;
                    p.probs[row] = (float)(weigh.weight(v[j]) * weigh.unit / (double)all);
                }
            }
        }
        if (__any_sync(kFullMask, here)) return;
        at_mass = shfl_idx(end_mass, 31);
        at_ties = (uint32_t)shfl_idx(end_ties, 31);
    }
}

}  // namespace

heph_status launch_sample(const SampleArgs &a, int sm_count, cudaStream_t stream) {
    // A row's blocks (a cluster) share its passes while there are fewer rows
    // than SMs and a block still has some work.
    uint32_t blocks = 1;
    while (blocks < kMaxCluster && (uint64_t)a.rows * blocks * 2 <= (uint32_t)sm_count && a.vocab / (blocks * 2) >= 4096)
        blocks *= 2;
    // vocab x 2^scale_bits stays below 2^62.
    const int bits = 32 - __builtin_clz(a.vocab);
    const SampleParams p{a.logits.ptr, a.logits.stride, a.uniform, a.temperature, a.top_p, a.min_p, a.top_k,
                         a.temperature_all, a.top_p_all, a.min_p_all, a.top_k_all, a.vocab, std::min(52, 62 - bits),
                         a.tokens, a.probs};
    return dispatch_row_dtype(a.dtype, [&]<typename T>() -> heph_status {
        HEPH_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           sizeof(SampleShared)),
                      HEPH_DISPATCH_FAILED, "token sampling shared memory");
        return launch_clusters("token sampling", sample_kernel<T>, dim3(a.rows * blocks), dim3(kSampleThreads), blocks,
                               sizeof(SampleShared), stream, p);
    });
}

}  // namespace heph
