// sample.cu — tokens drawn from rows of logits with temperature, top-k, top-p
// and min-p, from given uniform numbers.
//
//   w_i = exp((l_i - max) / T).  In the order of falling l (equal ones by
//   index): top-k keeps the first k; top-p of those the ones before which less
//   than p of their mass lies; min-p of those the ones of w >= min_p; the first
//   always stays.  The token is the first index whose running sum of kept w
//   exceeds u times the whole.
//
// Masses are whole numbers, w in units of 2^-scale_bits (44 for a vocabulary
// of 2^17), so that sums do not depend on their order: the answer is the same
// in any batch and for any number of blocks per row.
//
// A row (a few hundred KB, read from memory once and then from L2) belongs to
// a block, or to a cluster of blocks where there are few rows.  Each row takes
// the shortest way that its settings allow:
//   largest only    one pass for the maximum, one for its first index;
//   top-k           a histogram of the logits tells which can be among the
//                   first k; these (hardly more than k) are gathered and sorted
//                   in shared memory, where the rest is prefix sums;
//   top-p           the same with a histogram of masses;
//   neither         the masses of the warps' parts, and a walk through one;
//   top-k or top-p that leave over 1024  the threshold (a key, and how many of
//                   those equal to it) by histograms of ever narrower ranges,
//                   then as above.
#include <cooperative_groups.h>

#include <cfloat>

#include "row_ops.h"
#include "row_utils.cuh"

namespace heph {

namespace {

namespace cg = cooperative_groups;

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kBinBits = 10;
constexpr int kBins = 1 << kBinBits;
constexpr int kBinsPerThread = kBins / kSampleThreads;
constexpr int kListed = 1024;  // candidates that are sorted in shared memory
constexpr int kEach = kListed / kSampleThreads;
constexpr int kMaxCluster = 8;

struct SampleParams {
    const void *logits;
    int64_t stride;
    const float *uniform, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    double temperature_all, top_p_all, min_p_all;
    int32_t top_k_all;
    uint32_t rows, vocab;
    int scale_bits, limb_bits;
    bool deal;  // rows of long work first
    int64_t *tokens;
    float *probs;
};

// Masses in three limbs of `limb_bits`, which a block's sums of cannot
// overflow: three additions whose results nobody waits for, in any order.
// Counts are in the first.
struct Histogram {
    uint32_t limb[3][kBins];
};

// Everything that is kept: logits above `value`, and the first `ties` equal to it.
struct Threshold {
    float value;
    uint32_t ties;
};

struct SampleShared {
    Histogram hist[2];
    uint64_t list[kListed];  // candidates: not-key above index, so that they rise in the order of the choice
    uint64_t mass[kListed];  // of the sorted candidates
    uint64_t scan[kSampleWarps];
    uint64_t warp_mass[kSampleWarps];
    uint32_t warp_ties[kSampleWarps];
    uint64_t block_mass;  // this block's share of a sum, read by the cluster
    uint32_t block_ties;
    float block_max, block_sum;
    uint32_t block_count;
    double roots[16];
    uint32_t listed[2];  // entries in `list`, and in `mass` where that is the second list
    Threshold keep;
    uint32_t row;  // that is worked on
    uint32_t found_bin;
    uint64_t found_above, found_in;
};

__device__ __forceinline__ void add_mass(Histogram &h, uint32_t bin, uint64_t mass, int limb_bits) {
    const uint32_t mask = (1u << limb_bits) - 1;
    atomicAdd(&h.limb[0][bin], (uint32_t)mass & mask);
    atomicAdd(&h.limb[1][bin], (uint32_t)(mass >> limb_bits) & mask);
    atomicAdd(&h.limb[2][bin], (uint32_t)(mass >> 2 * limb_bits));
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

// Sum of v over the threads below, and over all; two barriers.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, SampleShared &s, uint64_t &all) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t upto = warp_scan(v);
    __syncthreads();
    if (lane == 31) s.scan[warp] = upto;
    __syncthreads();
    uint64_t below = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kSampleWarps; ++w) {
        below += w < (int)warp ? s.scan[w] : 0;
        all += s.scan[w];
    }
    return below + upto - v;
}

// One row, seen by one warp: the row's 16-byte vectors are cut into equal
// parts, so that blocks, warps, steps, lanes and elements follow the indices.
template <typename T> struct RowPart {
    static constexpr int V = 16 / sizeof(T);
    const T *row;
    const uint4 *vectors;  // the row's first vector, `lead` elements before it
    uint32_t vocab, lead;
    uint32_t begin, end;             // vectors of this warp
    uint32_t whole_begin, whole;     // of these, the ones that lie in the row: first, and how many

    __device__ RowPart(const T *row_, uint32_t vocab_, uint32_t parts, uint32_t part) : row(row_), vocab(vocab_) {
        lead = (uint32_t)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
        vectors = reinterpret_cast<const uint4 *>(row - lead);
        const uint32_t count = (lead + vocab + V - 1) / V;
        const uint32_t each = ((count + parts - 1) / parts + 31) / 32 * 32;
        begin = min(each * part, count);
        end = min(begin + each, count);
        whole_begin = begin + (begin == 0 && lead);
        const uint32_t whole_end = min(end, (lead + vocab) / V);
        whole = whole_end > whole_begin ? whole_end - whole_begin : 0;
    }
    // Vector q; what is outside the part or the row is NaN.
    __device__ __forceinline__ uint4 load(uint32_t q) const {
        if (q - whole_begin < whole) return vectors[q];
        if (q < end) return load_edge(q);
        return make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);  // a NaN in every type
    }
    __device__ __noinline__ uint4 load_edge(uint32_t q) const {
        Pack<T, V> u;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint32_t at = q * V + j - lead;  // wraps before the row
            u.e[j] = at < vocab ? row[at] : from_f32<T>(NAN);
        }
        return bitcast<uint4>(u);
    }
    // f(logits, index of the first) for every vector of the part; what is
    // outside is NaN.
    template <typename F> __device__ __forceinline__ void each(F &&f) const {
        uint32_t q = begin + (threadIdx.x & 31);
        uint4 a = load(q), b = load(q + 32);
#pragma unroll 1
        for (; q < end; q += 64) {
            const uint4 c = load(q + 64), d = load(q + 96);
            float u[V], v[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                u[j] = to_f32(bitcast<Pack<T, V>>(a).e[j]);
                v[j] = to_f32(bitcast<Pack<T, V>>(b).e[j]);
            }
            f(u, q * V - lead);
            f(v, (q + 32) * V - lead);
            a = c;
            b = d;
        }
    }
    // The same for short work, whose time is that of the loads: FAR of them at
    // once (two in each(); the passes for the maximum: 256 mixed rows 146 -> 140 us).
    template <int FAR, typename F> __device__ __forceinline__ void each_far(F &&f) const {
#pragma unroll 1
        for (uint32_t q = begin + (threadIdx.x & 31); q < end; q += 32 * FAR) {
            uint4 a[FAR];
#pragma unroll
            for (int i = 0; i < FAR; ++i) a[i] = load(q + 32 * i);
#pragma unroll
            for (int i = 0; i < FAR; ++i) {
                float u[V];
#pragma unroll
                for (int j = 0; j < V; ++j) u[j] = to_f32(bitcast<Pack<T, V>>(a[i]).e[j]);
                f(u, (q + 32 * i) * V - lead);
            }
        }
    }
    // f(logit, logit) for all elements, two at a time: for work so long that it
    // is written out once only (the instructions come from the cache too).
    template <typename F> __device__ __forceinline__ void each_two(F &&f) const {
        uint32_t q = begin + (threadIdx.x & 31);
        uint4 a = load(q), b = load(q + 32);
#pragma unroll 1
        for (; q < end; q += 32) {
            const uint4 c = load(q + 64);
#pragma unroll 1
            for (int i = 0; i < V / 2; ++i) {
                if constexpr (sizeof(T) == 4) {
                    f(__uint_as_float(a.x), __uint_as_float(a.y));
                    a.x = a.z;
                    a.y = a.w;
                } else {
                    const auto two = bitcast<Pack<T, 2>>(a.x);
                    f(to_f32(two.e[0]), to_f32(two.e[1]));
                    a.x = a.y;
                    a.y = a.z;
                    a.z = a.w;
                }
            }
            a = b;
            b = c;
        }
    }
};

// 2^(i / 16) by table, 2^(r / 16) for |r| <= 1/2 by the polynomial through the
// six Chebyshev nodes there, its constant being made 1: within 1e-14 together.
// (A table of 16 is 128 bytes of shared memory, one round of its banks.)
__constant__ double kRoots[16] = {
    0x1.0000000000000p+0, 0x1.0b5586cf9890fp+0, 0x1.172b83c7d517bp+0, 0x1.2387a6e756238p+0,
    0x1.306fe0a31b715p+0, 0x1.3dea64c123422p+0, 0x1.4bfdad5362a27p+0, 0x1.5ab07dd485429p+0,
    0x1.6a09e667f3bcdp+0, 0x1.7a11473eb0187p+0, 0x1.8ace5422aa0dbp+0, 0x1.9c49182a3f090p+0,
    0x1.ae89f995ad3adp+0, 0x1.c199bdd85529cp+0, 0x1.d5818dcfba487p+0, 0x1.ea4afa2a490dap+0};
__constant__ double kExp2[6] = {0x1.0000000000000p+0,  0x1.62e42fefa39f3p-5,  0x1.ebfbdff555824p-11,
                                0x1.c6b08d6f2a289p-17, 0x1.3b2c9b8a6caeap-23, 0x1.5d897e525c216p-30};

struct Weigher {
    float max, floor;  // floor: a lower logit has no mass
    float top, slope32;  // max, or the largest finite number; twice the slope in 32 bits
    double slope;        // 16 log2(e) / T
    int scale_bits, limb_bits;
    const double *roots;  // kRoots in shared memory

    __device__ Weigher(float max_, double t, int scale_bits_, int limb_bits_, const double *roots_)
        : max(max_), scale_bits(scale_bits_), limb_bits(limb_bits_), roots(roots_) {
        top = fminf(max, FLT_MAX);
        slope = 16 * 1.4426950408889634 / t;
        slope32 = (float)(2.0 * slope);
        // Below half a unit; and no -inf, whatever the temperature.  Rounded up:
        // the next number below may be thousands of T further down, where
        // mass() has no exponent for it.
        floor = fmaxf(__double2float_ru((double)max - (scale_bits + 1.5) * 0.6931471805599453 * t), -FLT_MAX);
    }
    // exp((l - max) / T) 2^scale_bits, rounded, for l >= floor (else anything);
    // a unit is at least 2^-45 of the maximum's mass, which is 2^scale_bits.
    __device__ __forceinline__ uint64_t mass(float l) const {
        l = fminf(l, FLT_MAX);  // an infinity is equal to itself
        // n = 16 log2(w) rounded, in the low bits of `at`.  From halves, as l -
        // top may pass the largest number.
        const float magic = 0x1.8p23f, at = fmaf(l, 0.5f, -0.5f * top) * slope32 + magic;
        const uint32_t n = __float_as_uint(at);
        const double r = fma((double)l - (double)top, slope, -(double)(at - magic));
        double p = kExp2[5];
#pragma unroll
        for (int i = 4; i >= 0; --i) p = fma(p, r, kExp2[i]);
        p *= roots[n & 15];
        // (n >> 4) + scale_bits more in the exponent; magic's own bits are shifted out.
        const double w = __hiloint2double(__double2hiint(p) + ((n & ~15u) << 16) + (scale_bits << 20), __double2loint(p));
        return (uint64_t)__double_as_longlong(w + 0x1p52) & 0xfffffffffffffull;
    }
    // The same unrounded, for the answer's probability.
    __device__ double share(float l, uint64_t all) const {
        const double w = l == max ? 1.0 : exp2(((double)l - (double)max) * (slope / 16));
        return ldexp(w, scale_bits) / (double)all;
    }
    __device__ __forceinline__ uint64_t mass_or_none(float l) const { return l >= floor ? mass(l) : 0; }
    // Of two at once, whose long chains of operations overlap.
    __device__ __forceinline__ void masses(float a, float b, float from, uint64_t &x, uint64_t &y) const {
        x = y = 0;
        if (a >= from || b >= from) {
            const uint64_t u = mass(a), v = mass(b);
            x = a >= from ? u : 0;
            y = b >= from ? v : 0;
        }
    }
};

// Which of 1024 equal steps below the maximum a logit is nearest to; the last
// takes all that is further down.  Falls monotonically in l.
struct Steps {
    float top, width;  // top is finite: +inf is in step 0 too
    float per_unit;
    __device__ Steps(const Weigher &weigh, float window) : top(weigh.top), width(window / kBins), per_unit(kBins / window) {}
    __device__ __forceinline__ uint32_t bin(float l) const {
        return __float_as_uint(fminf((top - l) * per_unit, (float)(kBins - 1)) + 0x1p23f) & (kBins - 1);
    }
    // No logit of step `bin` is above the one or below the other (a margin
    // covers the roundings of the step's number).
    __device__ float above(uint32_t bin) const {
        return bin ? __double2float_ru((double)top - (bin - 0.5) * width * (1.0 - 1e-6)) : INFINITY;
    }
    __device__ float below(uint32_t bin) const {
        return bin < kBins - 1 ? __double2float_rd((double)top - (bin + 0.5) * width * (1.0 + 1e-6)) : -INFINITY;
    }
};

template <int V> __device__ __forceinline__ float largest(const float (&v)[V]) {  // fmaxf passes NaN over
    float m = v[0];
#pragma unroll
    for (int j = 1; j < V; ++j) m = fmaxf(m, v[j]);
    return m;
}

// Sum of what `of` is in the blocks below `upto` of the cluster, by every warp.
template <typename N> __device__ __forceinline__ N sum_over_blocks(const N &of, uint32_t upto) {
    const uint32_t lane = threadIdx.x & 31;
    const cg::cluster_group cluster = cg::this_cluster();
    N v = 0;
    if (lane < upto) v = *cluster.map_shared_rank(&of, lane);
    return warp_fold<N, OP_SUM>(v);
}

__device__ __noinline__ void mass_to_bin(const Weigher &weigh, Histogram &h, uint32_t bin, float l) {
    const uint64_t mass = weigh.mass_or_none(l);
    if (mass) add_mass(h, bin, mass, weigh.limb_bits);
}

__device__ __forceinline__ void clear(Histogram &h) {
    for (int i = threadIdx.x; i < kBins; i += kSampleThreads) h.limb[0][i] = h.limb[1][i] = h.limb[2][i] = 0;
    __syncthreads();
}

// After a cluster barrier: the sums of the blocks' histograms, the first bin
// at which `before` plus the running sum reaches `wanted(all)` (kBins: none),
// what it holds, and the sum before it; the same for every block.
template <bool MASS, typename Wanted>
__device__ uint32_t find_bin(Histogram &h, SampleShared &s, int limb_bits, uint64_t before, Wanted &&wanted) {
    const cg::cluster_group cluster = cg::this_cluster();
    using Bins = Pack<uint32_t, kBinsPerThread>;
    const uint32_t t = threadIdx.x;
    uint64_t bins[kBinsPerThread] = {}, sum = 0, all;
#pragma unroll
    for (int limb = 0; limb < (MASS ? 3 : 1); ++limb) {
        Bins theirs[kMaxCluster] = {};
#pragma unroll
        for (uint32_t b = 0; b < kMaxCluster; ++b)
            if (b < cluster.num_blocks())
                theirs[b] = *reinterpret_cast<const Bins *>(&cluster.map_shared_rank(&h, b)->limb[limb][t * kBinsPerThread]);
#pragma unroll
        for (int i = 0; i < kBinsPerThread; ++i) {
            uint64_t of = 0;
#pragma unroll
            for (int b = 0; b < kMaxCluster; ++b) of += theirs[b].e[i];
            bins[i] += of << limb * limb_bits;
        }
    }
#pragma unroll
    for (int i = 0; i < kBinsPerThread; ++i) sum += bins[i];
    if (t == 0) s.found_bin = kBins;
    uint64_t run = before + block_scan(sum, s, all);
    const uint64_t goal = wanted(all);
#pragma unroll
    for (int i = 0; i < kBinsPerThread; ++i) {
        if (run < goal && run + bins[i] >= goal) {
            s.found_bin = t * kBinsPerThread + i;
            s.found_above = run;
            s.found_in = bins[i];
        }
        run += bins[i];
    }
    __syncthreads();
    return s.found_bin;
}

// The step of the logit in which a search is known to end.
struct Located {
    uint32_t bin = kBins;  // not known
    uint64_t above = 0, wanted = 0;
};

struct Narrowed {
    uint32_t key;    // 0: the row's keys above the floor do not reach it
    uint64_t above;  // count or mass of the keys above `key`, or of all
    uint64_t wanted;
};

// The largest key such that the keys at or above it hold at least wanted =
// need(total) (a count, or with MASS a mass), among the row's logits above
// `floor`, of which `total` is the whole.  First by steps of the logit below
// the maximum, which spreads any scale of logits; then, within one of them,
// by steps of the key.
template <bool MASS, typename T, typename Need>
__device__ Narrowed narrow(const RowPart<T> &part, const Weigher &weigh, SampleShared &s, int &turn, float floor,
                           float window, const Located &start, Need &&need) {
    const cg::cluster_group cluster = cg::this_cluster();
    const Steps steps(weigh, window);
    Narrowed got{0, start.above, start.wanted};
    uint32_t first = start.bin, high = ordered_key(weigh.max), low = 1;
    int shift = -1;  // -1: steps of the logit
    // The keys that step `first` may have; which of them belong is decided by
    // their step's number.
    auto enter_step = [&] {
        high = ::min(high, ordered_key(steps.above(first)));
        low = ::max(low, ordered_key(steps.below(first)));
    };
    if (first < kBins) {
        enter_step();
        shift = ::max(0, 32 - __clz(high - low) - kBinBits);
    }
    for (;;) {
        Histogram &h = s.hist[turn];
        turn ^= 1;
        clear(h);
        // Logits that may be counted now; all others are passed over.  Whether a
        // logit is between the keys is asked of its own key: 0x7fffffff is no
        // number's (both zeros have 0x80000000), and as a float it is -0.
        const float from = shift < 0 ? floor : key_value(low);
        part.each([&](const float(&v)[RowPart<T>::V], uint32_t) {
            if (!(largest(v) >= from)) return;
#pragma unroll
            for (int j = 0; j < RowPart<T>::V; ++j) {
                const float l = v[j];
                if (!(l >= from && l > floor)) continue;
                uint32_t bin = steps.bin(l);
                if (shift >= 0) {
                    const uint32_t key = ordered_number(l);
                    if (bin != first || key < low || key > high) continue;
                    bin = (high - key) >> shift;
                }
                if constexpr (MASS) mass_to_bin(weigh, h, bin, l);
                else atomicAdd(&h.limb[0][bin], 1u);
            }
        });
        cluster.sync();
        // The other histogram is cleared next, after this barrier, when no
        // block reads it any more.
        uint64_t total = 0;
        const uint32_t bin = find_bin<MASS>(h, s, weigh.limb_bits, got.above, [&](uint64_t all) {
            total = all;
            if (shift < 0) got.wanted = need(all);
            return got.wanted;
        });
        if (bin == kBins) {
            got.above = total;
            return got;
        }
        got.above = s.found_above;
        if (shift < 0) {
            first = bin;
            enter_step();
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

// Sorts `size` (a power of two) numbers upwards; a small list by one warp.
__device__ void sort_list(uint64_t *list, uint32_t size) {
    const uint32_t warp = threadIdx.x >> 5;
    const bool small = size <= 64;
    if (!small || warp == 0) {
        for (uint32_t run = 2; run <= size; run *= 2) {
            for (uint32_t d = run / 2; d > 0; d /= 2) {
                for (uint32_t i = threadIdx.x; i < size / 2; i += kSampleThreads) {
                    const uint32_t a = 2 * i - (i & (d - 1)), b = a + d;
                    const uint64_t x = list[a], y = list[b];
                    if ((x > y) == ((a & run) == 0)) {
                        list[a] = y;
                        list[b] = x;
                    }
                }
                if (small) __syncwarp();
                else __syncthreads();
            }
        }
    }
    __syncthreads();
}

__device__ __forceinline__ uint32_t power_from(uint32_t n) { return n <= 2 ? 2 : 1u << (32 - __clz(n - 1)); }

__device__ __forceinline__ uint64_t part_of(uint64_t all, double p) {  // ceil(p all), from 1 to all
    const double part = ceil((double)all * (p > 0.0 ? p : 0.0));
    return part < 1.0 ? 1 : ::min((uint64_t)part, all);
}
__device__ __forceinline__ uint64_t point_of(uint64_t all, float u) {  // floor(u all), below all
    return ::min((uint64_t)((u > 0.0f ? (double)fminf(u, 1.0f) : 0.0) * (double)all), all - 1);
}

// Block 0 gathers the cluster's lists (which = 1: the second) in s.list; its
// length.  Warp b fetches block b's.
__device__ uint32_t collect(SampleShared &s, int which) {
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t warp = threadIdx.x >> 5, blocks = cluster.num_blocks();
    if (cluster.block_rank() == 0 && warp < blocks && (warp || which)) {
        const uint32_t to = sum_over_blocks(s.listed[which], warp);
        const SampleShared *o = cluster.map_shared_rank(&s, warp);
        const uint64_t *list = which ? o->mass : o->list;
        for (uint32_t i = threadIdx.x & 31; i < o->listed[which]; i += 32) s.list[to + i] = list[i];
    }
    return sum_over_blocks(s.listed[which], blocks);
}

// s.list sorted upwards, n entries and padding; this thread's kEach of them
// (0 past n).
__device__ void sorted_entries(SampleShared &s, uint32_t n, uint64_t (&entry)[kEach]) {
    const uint32_t t = threadIdx.x, size = power_from(n);
    for (uint32_t i = n + t; i < size; i += kSampleThreads) s.list[i] = ~0ull;
    __syncthreads();
    sort_list(s.list, size);
#pragma unroll
    for (int i = 0; i < kEach; ++i) entry[i] = t * kEach + i < n ? s.list[t * kEach + i] : 0;
}

__device__ __forceinline__ float entry_logit(uint64_t entry) { return key_value(~(uint32_t)(entry >> 32)); }

// The threshold that is known to lie among the n entries of s.list, all there
// are of their step of the logit.  One block.
__device__ void threshold_from_list(const Weigher &weigh, SampleShared &s, uint32_t n, bool count, const Located &located) {
    uint64_t entry[kEach], size[kEach], sum = 0, all;
    sorted_entries(s, n, entry);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        size[i] = threadIdx.x * kEach + i >= n ? 0 : count ? 1 : weigh.mass_or_none(entry_logit(entry[i]));
        sum += size[i];
    }
    uint64_t run = located.above + block_scan(sum, s, all);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        if (run < located.wanted && run + size[i] >= located.wanted) {
            // The last that is kept; the ones equal to it stand before it.
            const uint32_t r = threadIdx.x * kEach + i;
            uint32_t first = r;
            while (first > 0 && s.list[first - 1] >> 32 == entry[i] >> 32) --first;
            s.keep = {entry_logit(entry[i]), r - first + 1};
        }
        run += size[i];
    }
}

// Draws from the n candidates in s.list, the row's first n (or more, in no
// order): the first k of them, of these the top-p of `whole` mass (0: of their
// own), of these those of mass >= least.  One block.
template <typename T>
__device__ void draw_from_list(const T *row, const Weigher &weigh, SampleShared &s, uint32_t n, uint32_t k, double top_p, uint64_t whole,
                               uint64_t least, float u, int64_t *token, float *prob) {
    const uint32_t t = threadIdx.x, of = min(n, k);
    uint64_t mass[kEach], entry[kEach], sum = 0, all;
    sorted_entries(s, n, entry);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        mass[i] = t * kEach + i < of ? weigh.mass_or_none(entry_logit(entry[i])) : 0;
        sum += mass[i];
    }
    uint64_t run = block_scan(sum, s, all);
    const uint64_t wanted = top_p < 1.0 ? part_of(whole ? whole : all, top_p) : ~0ull;
    bool keep[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const uint32_t r = t * kEach + i;
        keep[i] = r < of && run < wanted && (mass[i] >= least || r == 0);
        run += mass[i];
        if (r < kListed) s.mass[r] = mass[i];
    }
    uint32_t kept = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) kept += __syncthreads_count(keep[i]);
    // The kept ones by index, and their running sum.
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const uint32_t r = t * kEach + i;
        if (r < kept) s.list[r] = entry[i] << 32 | r;
    }
    __syncthreads();
    sorted_entries(s, kept, entry);
    sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        mass[i] = t * kEach + i < kept ? s.mass[(uint32_t)entry[i]] : 0;
        sum += mass[i];
    }
    run = block_scan(sum, s, all);
    const uint64_t point = point_of(all, u);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        if (point >= run && point < run + mass[i]) {
            *token = (int64_t)(entry[i] >> 32);
            *prob = (float)weigh.share(to_f32(row[entry[i] >> 32]), all);
        }
        run += mass[i];
    }
}

// What a row asks for.
struct Asked {
    double t, top_p;
    int32_t k;
    bool greedy, by_count, by_mass;
    __device__ Asked(const SampleParams &p, uint32_t row)
        : t(p.temperature ? p.temperature[row] : p.temperature_all), top_p(p.top_p ? p.top_p[row] : p.top_p_all),
          k(p.top_k ? p.top_k[row] : p.top_k_all) {
        greedy = !(t > 0.0) || k == 1;
        by_count = !greedy && k > 0 && (uint32_t)k < p.vocab;
        by_mass = !greedy && top_p < 1.0;
    }
    // Most work first.
    __device__ __forceinline__ uint32_t order() const { return by_mass && !by_count ? 0 : greedy ? 2 : 1; }
};

// The row that is `place`-th by order(), then by index; of at most
// kSampleThreads rows, a thread each.
__device__ uint32_t dealt_row(const SampleParams &p, SampleShared &s, uint32_t place) {
    const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const uint32_t order = t < p.rows ? Asked(p, t).order() : 3;
    const uint32_t first = __syncthreads_count(order == 0), second = __syncthreads_count(order == 1);
    const uint32_t alike = __match_any_sync(kFullMask, order);
    // Rows of each order in the warps below, ten bits each.
    if (lane == 0) s.scan[warp] = 0;
    __syncwarp();
    if (order < 3 && lane == __ffs(alike) - 1u) atomicAdd((unsigned long long *)&s.scan[warp], (unsigned long long)__popc(alike) << order * 10);
    __syncthreads();
    uint64_t below = 0;
#pragma unroll
    for (int w = 0; w < kSampleWarps; ++w) below += w < (int)warp ? s.scan[w] : 0;
    const uint32_t at = (order > 0 ? first : 0) + (order > 1 ? second : 0) + (uint32_t)(below >> (order * 10) & 1023u) +
                        __popc(alike & ((1u << lane) - 1));
    if (order < 3 && at == place) s.row = t;
    __syncthreads();
    return s.row;
}

// Two blocks an SM leave 64 registers a thread, of which 216 bytes are spilled
// (reads of 248, f32 336).  Bound by the latency of its chains of dependent
// operations (four warps a scheduler in a block) and, where it searches a
// threshold, by the block's barriers: 128 x 50257 bf16 at temperature alone has
// 43 % of its issue slots filled and 12 % of the fp64 pipe, 256 x 131072 f32 60 %
// and 18 %, with top-p 64 % and 13 %.
template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const __grid_constant__ SampleParams p) {
    __shared__ SampleShared s;
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t blocks = cluster.num_blocks(), block = cluster.block_rank();
    const uint32_t row = p.deal ? dealt_row(p, s, blockIdx.x / blocks) : blockIdx.x / blocks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const RowPart<T> part(static_cast<const T *>(p.logits) + row * p.stride, p.vocab, blocks * kSampleWarps,
                          block * kSampleWarps + warp);
    const Asked asked(p, row);
    double t = asked.t;
    const int32_t k = asked.k;
    const double top_p = asked.top_p;
    const double min_p = p.min_p ? p.min_p[row] : p.min_p_all;
    const float u = p.uniform[row];
    const bool greedy = asked.greedy, by_count = asked.by_count, by_mass = asked.by_mass;

    // The maximum, and for top-k the mean, which tells the logits' scale.
    float max = -INFINITY, sum = 0.0f;
    uint32_t count = 0;
    part.template each_far<8>([&](const float(&v)[RowPart<T>::V], uint32_t) {
        max = fmaxf(max, largest(v));
        if (fabsf(v[0]) < 1e4f) {  // of every V-th; no masks
            sum += v[0];
            ++count;
        }
    });
    max = warp_max(max);
    sum = warp_sum(sum);
    count = warp_fold<uint32_t, OP_SUM>(count);
    if (lane == 0) {
        s.warp_mass[warp] = (uint64_t)__float_as_uint(max) << 32 | __float_as_uint(sum);
        s.warp_ties[warp] = count;
    }
    if (threadIdx.x < 2) s.listed[threadIdx.x] = 0;
    if (threadIdx.x < 16) s.roots[threadIdx.x] = kRoots[threadIdx.x];
    __syncthreads();
    if (warp == 0) {
        const bool has = lane < kSampleWarps;
        const uint64_t both = has ? s.warp_mass[lane] : 0;
        max = warp_max(has ? __uint_as_float((uint32_t)(both >> 32)) : -INFINITY);
        sum = warp_sum(has ? __uint_as_float((uint32_t)both) : 0.0f);
        count = warp_fold<uint32_t, OP_SUM>(has ? s.warp_ties[lane] : 0);
        if (lane == 0) {
            s.block_max = max;
            s.block_sum = sum;
            s.block_count = count;
        }
    }
    cluster.sync();
    max = warp_max(lane < blocks ? *cluster.map_shared_rank(&s.block_max, lane) : -INFINITY);
    sum = sum_over_blocks(s.block_sum, blocks);
    count = sum_over_blocks(s.block_count, blocks);
    if (max == -INFINITY) {  // nothing to choose from
        if (block == 0 && threadIdx.x == 0) {
            p.tokens[row] = -1;
            p.probs[row] = 0.0f;
        }
        cluster.sync();
        return;
    }
    if (greedy) {
        uint32_t first = ~0u;
        part.template each_far<8>([&](const float(&v)[RowPart<T>::V], uint32_t index) {
#pragma unroll
            for (int j = 0; j < RowPart<T>::V; ++j)
                if (v[j] == max) first = min(first, index + j);
        });
        first = warp_fold<uint32_t, OP_MIN>(first);
        if (lane == 0) s.warp_ties[warp] = first;
        __syncthreads();
        if (warp == 0) {
            first = warp_fold<uint32_t, OP_MIN>(lane < kSampleWarps ? s.warp_ties[lane] : ~0u);
            if (lane == 0) s.block_ties = first;
        }
        cluster.sync();
        if (block == 0 && threadIdx.x == 0) {
            for (uint32_t b = 1; b < blocks; ++b) first = min(first, *cluster.map_shared_rank(&s.block_ties, b));
            p.tokens[row] = first;
            p.probs[row] = 1.0f;
        }
        cluster.sync();
        return;
    }

    t = fmax(t, 0x1p-100);  // 1 / t stays a number in 32 bits
    const Weigher weigh(max, t, p.scale_bits, p.limb_bits, s.roots);
    const double least_w = min_p > 0.0 ? fmin(min_p, 1.0) : 0.0;
    const uint64_t least = (uint64_t)ceil(least_w * (double)(1ull << p.scale_bits));
    // top-k: the distance from the mean to the maximum covers every k below
    // half of the vocabulary, and three quarters of it a k below an eighth (of
    // normal logits; others are found too, the longer way).  top-p: what is left below the window is less
    // than 1 - p of the mass, were it all as heavy as its upper end.
    const float spread = (count && max < 1e4f ? max - sum / count : 16.0f) * ((uint32_t)k < p.vocab / 8 ? 0.75f : 1.0f);
    const float count_window = fminf(fmaxf(spread, 0x1p-10f), 0x1p10f);
    const float mass_window =
        fminf(fmaxf((float)t * (__logf((float)p.vocab / fmaxf((float)(1.0 - top_p), 1e-6f)) + 0.01f), 0x1p-10f), 0x1p10f);
    int turn = 0;
    Located located;
    Threshold keep{-INFINITY, 0};
    bool found = false;

    if (by_count || by_mass) {
        Histogram &h = s.hist[turn];
        uint32_t last = kBins - 1;
        bool fits = p.vocab <= kListed;  // all that is kept may fit a list
        uint64_t whole = 0;
        const Steps steps(weigh, by_count ? count_window : mass_window);
        const float edge = steps.top - (by_count ? count_window : mass_window);
        if (!fits) {
            turn ^= 1;
            clear(h);
        }
        if (fits) {
            // All of it is listed.
        } else if (by_count) {
            part.template each_far<4>([&](const float(&v)[RowPart<T>::V], uint32_t) {
                if (!(largest(v) >= edge)) return;
#pragma unroll
                for (int j = 0; j < RowPart<T>::V; ++j)
                    if (v[j] >= edge) atomicAdd(&h.limb[0][steps.bin(v[j])], 1u);
            });
            cluster.sync();
            last = find_bin<false>(h, s, 0, 0, [&](uint64_t) { return (uint64_t)k; });
            if (last < kBins - 1) located = {last, s.found_above, (uint64_t)k};
            fits = located.bin < kBins && s.found_above + s.found_in <= kListed;
        } else {
            uint64_t mass = 0;
            part.each_two([&](float a, float b) {
                uint64_t x, y;
                weigh.masses(a, b, weigh.floor, x, y);
                mass += x + y;
                if (a >= edge) add_mass(h, steps.bin(a), x, weigh.limb_bits);
                if (b >= edge) add_mass(h, steps.bin(b), y, weigh.limb_bits);
            });
            uint64_t mine;
            block_scan(mass, s, mine);
            if (threadIdx.x == 0) s.block_mass = mine;
            cluster.sync();
            whole = (uint64_t)sum_over_blocks((int64_t &)s.block_mass, blocks);
            last = find_bin<true>(h, s, weigh.limb_bits, 0, [&](uint64_t) { return part_of(whole, top_p); });
            fits = last < kBins - 1;
            if (fits) located = {last, s.found_above, part_of(whole, top_p)};
        }
        if (fits || located.bin < kBins) {
            // Two lists: of all that may be kept, and of the last step alone.
            const float from = steps.below(last), above = steps.above(last);
            part.each([&](const float(&v)[RowPart<T>::V], uint32_t index) {
                if (!(largest(v) >= from)) return;
                // Past its end the first list is of no use, and a common counter slow.
                const bool both = fits && *(volatile uint32_t *)&s.listed[0] <= kListed;
                const float upto = both ? INFINITY : above;
#pragma unroll
                for (int j = 0; j < RowPart<T>::V; ++j) {
                    if (!(v[j] >= from && v[j] <= upto)) continue;
                    const uint32_t bin = steps.bin(v[j]);
                    const uint64_t entry = (uint64_t)~ordered_number(v[j]) << 32 | (index + j);
                    if (both && bin <= last) {
                        const uint32_t at = atomicAdd(&s.listed[0], 1u);
                        if (at < kListed) s.list[at] = entry;
                    }
                    if (bin == last) {
                        const uint32_t at = atomicAdd(&s.listed[1], 1u);
                        if (at < kListed) s.mass[at] = entry;
                    }
                }
            });
            cluster.sync();
            if (fits && sum_over_blocks(s.listed[0], blocks) <= kListed) {
                const uint32_t n = collect(s, 0);
                cluster.sync();
                if (block == 0)
                    draw_from_list(part.row, weigh, s, n, by_count ? k : n, top_p, whole, least, u, p.tokens + row, p.probs + row);
                return;
            }
            if (sum_over_blocks(s.listed[1], blocks) <= kListed) {
                const uint32_t n = collect(s, 1);
                if (block == 0) threshold_from_list(weigh, s, n, by_count, located);
                cluster.sync();
                keep = *cluster.map_shared_rank(&s.keep, 0);
                found = true;
            }
        }
    }

    // The threshold, where top-k or top-p have it left to be found.
    if (by_count && !found) {
        const Narrowed n = narrow<false>(part, weigh, s, turn, -INFINITY, count_window, located, [&](uint64_t) { return (uint64_t)k; });
        if (n.key) keep = {key_value(n.key), (uint32_t)(k - n.above)};
    }
    if (by_mass && (by_count || !found)) {
        const uint64_t tie = keep.ties ? weigh.mass_or_none(keep.value) : 0;
        const Narrowed n = narrow<true>(part, weigh, s, turn, keep.value, mass_window, by_count ? Located{} : located,
                                        [&](uint64_t above) { return part_of(above + keep.ties * tie, top_p); });
        // What is left to be filled by logits equal to the key's.
        const uint64_t left = n.wanted - n.above, each = n.key ? weigh.mass_or_none(key_value(n.key)) : tie;
        const uint32_t ties = each ? (uint32_t)((left + each - 1) / each) : 0;
        keep = {n.key ? key_value(n.key) : keep.value, ties};
    }

    // Kept mass and ties, per warp, block and row.
    float from = weigh.floor;  // no lower logit is kept
    if (least_w > 0.0) from = fmaxf(from, __double2float_rd((double)max + t * (log(least_w) - 1e-9)));
    if (keep.value >= from) from = keep.value < INFINITY ? nextafterf(keep.value, INFINITY) : NAN;  // NAN: none is above
    auto kept_masses = [&](float a, float b, uint64_t &x, uint64_t &y) {
        weigh.masses(a, b, from, x, y);
        x = x >= least ? x : 0;
        y = y >= least ? y : 0;
    };
    uint64_t tie = keep.ties ? weigh.mass_or_none(keep.value) : 0;
    if (tie < least) tie = 0;
    uint64_t mass = 0;
    uint32_t ties = 0;
    if (keep.ties == 0 && least == 0) {
        part.each_two([&](float a, float b) {
            uint64_t x, y;
            weigh.masses(a, b, from, x, y);
            mass += x + y;
        });
    } else {
        part.each_two([&](float a, float b) {
            uint64_t x, y;
            kept_masses(a, b, x, y);
            mass += x + y;
            ties += (a == keep.value) + (b == keep.value);
        });
    }
    mass = warp_fold<int64_t, OP_SUM>((int64_t)mass);
    ties = warp_fold<uint32_t, OP_SUM>(ties);
    if (lane == 0) {
        s.warp_mass[warp] = mass;
        s.warp_ties[warp] = ties;
    }
    __syncthreads();
    if (warp == 0) {
        const uint64_t m = warp_fold<int64_t, OP_SUM>(lane < kSampleWarps ? (int64_t)s.warp_mass[lane] : 0);
        const uint32_t n = warp_fold<uint32_t, OP_SUM>(lane < kSampleWarps ? s.warp_ties[lane] : 0);
        if (lane == 0) {
            s.block_mass = m;
            s.block_ties = n;
        }
    }
    cluster.sync();
    auto kept = [&](uint64_t m, uint64_t n) { return m + (n < keep.ties ? n : keep.ties) * tie; };
    const uint64_t all = kept((uint64_t)sum_over_blocks((int64_t &)s.block_mass, blocks), sum_over_blocks(s.block_ties, blocks));
    uint64_t at_mass = (uint64_t)sum_over_blocks((int64_t &)s.block_mass, block);
    uint32_t at_ties = sum_over_blocks(s.block_ties, block);
    cluster.sync();  // the last reads of other blocks' memory
    const uint64_t point = point_of(all, u);
    // The block in whose part the running sum passes the point walks through
    // the part of its warp in which it does, a vector a thread.
    if (point < kept(at_mass, at_ties)) return;
    const uint64_t warps_mass = lane < kSampleWarps ? s.warp_mass[lane] : 0, upto_mass = warp_scan(warps_mass);
    const uint32_t warps_ties = lane < kSampleWarps ? s.warp_ties[lane] : 0, upto_ties = (uint32_t)warp_scan(warps_ties);
    const uint32_t past = __ballot_sync(kFullMask, point < kept(at_mass + upto_mass, at_ties + upto_ties));
    if (!past) return;
    const uint32_t owner = __ffs(past) - 1;
    at_mass += shfl_idx(upto_mass - warps_mass, owner);
    at_ties += shfl_idx(upto_ties - warps_ties, owner);
    const RowPart<T> theirs(part.row, p.vocab, blocks * kSampleWarps, block * kSampleWarps + owner);
    for (uint32_t q0 = theirs.begin; q0 < theirs.end; q0 += kSampleThreads) {
        constexpr int V = RowPart<T>::V;
        const uint32_t q = q0 + threadIdx.x;
        const auto v = bitcast<Pack<T, V>>(theirs.load(q));
        uint64_t m[V], step_mass = 0, more_mass, more_ties;
        uint32_t n = 0;
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            kept_masses(to_f32(v.e[j]), to_f32(v.e[j + 1]), m[j], m[j + 1]);
            step_mass += m[j] + m[j + 1];
            n += (to_f32(v.e[j]) == keep.value) + (to_f32(v.e[j + 1]) == keep.value);
        }
        uint64_t run_mass = at_mass + block_scan(step_mass, s, more_mass), run_ties = at_ties + block_scan(n, s, more_ties);
        at_mass += more_mass;
        at_ties += (uint32_t)more_ties;
        if (point < kept(run_mass + step_mass, run_ties + n) && point >= kept(run_mass, run_ties)) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float l = to_f32(v.e[j]);
                const uint64_t before = kept(run_mass, run_ties);
                run_mass += m[j];
                run_ties += l == keep.value;
                if (point >= before && point < kept(run_mass, run_ties)) {
                    p.tokens[row] = (int64_t)q * V - part.lead + j;
                    p.probs[row] = (float)weigh.share(l, all);
                }
            }
        }
        if (point < kept(at_mass, at_ties)) return;
    }
}

}  // namespace

heph_status launch_sample(const SampleArgs &a, int sm_count, cudaStream_t stream) {
    // A row's blocks (a cluster) share its passes: as many as there are SMs
    // for all rows, while each still has some work; and, as rows may differ
    // much in theirs, never over a share of 64 K logits each.  Measured on one
    // B200 with 1 / 2 / 4 / 8 blocks a row: 1 row of 131072 41 / 29 / 22 / 21
    // us, 128 of 50257 27 / 31 / 43 / 65, 256 of 131072, each with settings of
    // its own and in the order of their index, 233 / 173 / 167 / 226.
    uint32_t blocks = 1;
    while (blocks < kMaxCluster && (((uint64_t)a.rows * blocks * 2 <= (uint32_t)sm_count && a.vocab / (blocks * 2) >= 4096) ||
                                    a.vocab / blocks >= 65536))
        blocks *= 2;
    // Rows that differ in their work and do not all run at once: the longest
    // start first, or they end alone.  Top-p rows take 3 to 5 times as long as
    // greedy ones: 256 of 131072 take 163 us in the order of their index, 150 in that of
    // their work.  Each block finds its row itself, from the settings (where all
    // are alike, 118 us instead of 115).  A thread looks at one row's, so batches past 512
    // rows stay in the order of their index: 512 of 131072 294 us, 513 314.
    const bool deal = (a.temperature || a.top_p || a.top_k) && (uint64_t)a.rows * blocks > 2 * (uint32_t)sm_count &&
                      a.rows <= kSampleThreads;
    // vocab x 2^scale_bits stays below 2^62, a mass below that of three limbs,
    // and the sum of a limb of a block's logits (an eighth of the row and 4096,
    // or less than 2^17) below 2^32.
    const int bits = 32 - __builtin_clz(a.vocab), limb_bits = a.vocab <= (1u << 20) - (1u << 16) ? 15 : 13;
    const SampleParams p{a.logits.ptr, a.logits.stride, a.uniform, a.temperature, a.top_p, a.min_p, a.top_k,
                         a.temperature_all, a.top_p_all, a.min_p_all, a.top_k_all, a.rows, a.vocab,
                         std::min(3 * limb_bits - 1, 62 - bits), limb_bits, deal, a.tokens, a.probs};
    return dispatch_row_dtype(a.dtype, [&]<typename T>() -> heph_status {
        return launch_clusters("token sampling", sample_kernel<T>, dim3(a.rows * blocks), dim3(kSampleThreads), blocks, 0,
                               stream, p);
    });
}

}  // namespace heph
