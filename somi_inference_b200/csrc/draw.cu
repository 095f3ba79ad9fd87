// Tokens drawn from rows of logits with the caller's uniform numbers: temperature, top-k, top-p, min-p, any
// number of draws a row.
//
//     w_i = 2^((x_i - max x) log2(e) / T), and nothing where it is below 2^-44
//     order: value descending, equal values by index.  top-k: the first k.  top-p: of what top-k left,
//     those with (mass in front) <= top_p (mass of what top-k left).  min-p: those with w_i >= min_p.
//     draw: the first i in index order whose cumulated mass over kept tokens is above u (kept mass)
//
// Which token a number falls on, and where a cut lies, is a comparison of sums, so these must not depend
// on the order of summation nor on float32's rounding: a weight is computed in float64 (2^r by its Taylor
// series, relative error 3e-16) and held as an integer multiple of 2^-44, and sums of integers are exact.
// (Fewer than 2^20 weights of at most 2^44 stay below 2^64.)  So the result is the same bits whatever the launch
// looks like, and differs from real arithmetic only where a border lies within n 2^-45 of the number, n the tokens with a
// weight, in units of the largest weight: 4e-9 for 152,064 tokens whose roundings all have one sign.
//
// A cluster of CTAs shares a row; each holds its slice in shared memory, read from HBM once, as a bulk copy where
// the row is aligned.  A warp owns a contiguous segment of it.  All three cuts keep a beginning of one order, so a
// token can be left out as soon as it is known to lie behind a cut:
//     top-k: the r-th largest of a CTA's warps' (or threads') maxima, r = k / (CTAs of the cluster), has r logits at or above
//            it in that CTA, so the least such value of the cluster has k at or above it in the row;
//     top-p: the masses of 2,048 bins of the logits' distance from the maximum say in which bin the cut lies;
//     min-p: by its definition.
// What is left (the survivors, in the order of their indices) is usually a few dozen to a few hundred tokens; they are
// collected in one CTA, sorted, cut and drawn from there: a row of 152,064 logits costs a pass for its maximum and one that
// looks for survivors, and only a row with top-p and without top-k a weight for every token.  Where more than
// `kListed` survive, the cuts are found by histograms that the cluster's CTAs add up: first those bins (they
// span the 30.5 temperatures in which weights do not vanish), then the keys (the order-preserving integer image of a
// float) that lie in the bin of the cut, until a bin is one key (top-p's bin, where it holds no more than `kListed`,
// is sorted in one CTA instead); what is kept is then a key and an index up to which logits equal to it are kept, and
// weights are computed a second time to find where the numbers fall (where top-p's bin was sorted, the bins above it tell every CTA
// what it keeps, and only one on which a number falls weighs again).
//
// Measured (152,064 logits): 1 row with all filters 11.1 us (a chain of exchanges and a sort; HBM would need 0.1), 8 rows without
// any 13.6, 64 rows of mixed settings 61 (57.5 in a graph; about 90 instructions a weight and token), 256 bfloat16 rows with top-p 217 (weighed once a
// value, 281 once a token): instructions at 2.1 of 4 issue slots a cycle, and barriers.
#include <cooperative_groups.h>

#include <algorithm>
#include <utility>

#include "mma.cuh"
#include "tma.cuh"

namespace somi {
namespace draw {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 1024, kMaxCluster = 16;
constexpr int kMassBins = 2048;              // of the masses that top-p cuts
constexpr int kListed = 2048;                // survivors that one CTA takes
constexpr int kBinListed = 1024;             // tokens of top-p's bin that one CTA takes
constexpr int kCounted = 2 * 16 * 128;       // values of 16-bit logits that are counted: signs, exponents (2^-8 to 2^8), mantissas
constexpr unsigned kCountedFrom = 119u << 7;
constexpr int kMostSlice = 192 * 1024;       // bytes of a slice beside the static shared memory
constexpr int kFraction = 44;                // a weight is an integer multiple of 2^-44
typedef unsigned long long u64;

struct Settings {
    const float *temperature, *top_p, *min_p, *penalty;
    const int *top_k, *hist_off, *hist_tok;
};

struct Token { unsigned key; int at; };

struct Shared {
    union {
        u64 hist[2][kBins];                  // (read by the other CTAs of the cluster)
        unsigned pieces[3][kMassBins];       // masses of bins in pieces of 15 bits (likewise)
        struct {
            union {
                Token list[kListed];         // this CTA's survivors (likewise)
                u64 bin_order[kBinListed];   // in the first CTA, where it cuts top-p's bin: its tokens by value and index
            };
            Token bin_list[kBinListed];      // this CTA's tokens of top-p's bin, in any order (read by the others)
        };
    };
    u64 scan[kWarps];
    u64 warp_sum[kWarps];
    u64 total[kMaxCluster], mass[kMaxCluster];   // written by the other CTAs, one exchange each
    unsigned top_key[kMaxCluster], floor_key[kMaxCluster], top_at[kMaxCluster], ties[kMaxCluster];
    uint2 listed[kMaxCluster];               // survivors, tokens of the cut's bin
    unsigned key[kWarps], at[kWarps];
    u64 cross_above, cross_mass;
    int cross_bin, tie_cut;
    unsigned bin_count;                      // of bin_list; more than it holds: some are missing
    unsigned cut_key;
    unsigned lo, hi;
    unsigned long long loaded;               // mbarrier of the bulk copy
};

__device__ int g_draw_error = 0;

__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
// A logit: NaN counts as -inf, -0 as 0 (equal values must have equal keys).
__device__ __forceinline__ float logit_of(float x) { return x == x ? x + 0.0f : -INFINITY; }

// ln(2)^K / K!
template <int K>
struct Taylor { static constexpr double value = Taylor<K - 1>::value * 0.69314718055994530942 / K; };
template <>
struct Taylor<0> { static constexpr double value = 1.0; };

// 2^r by the first N + 1 terms of its Taylor series, |r| <= 1/2 (N = 12: 2e-16)
template <int N, int K = 0>
__device__ __forceinline__ double exp2_taylor(double r) {
    if constexpr (K == N) return Taylor<K>::value;
    else return fma(exp2_taylor<N, K + 1>(r), r, Taylor<K>::value);
}

// A row's maximum and temperature: what a weight depends on.
struct Heat {
    float top;
    double c;                                // log2(e) / T
    float bins;                              // 1 / the distance from the maximum at which bins end

    // w 2^44 before it is rounded to an integer; 0 where w < 2^-44.  NaN and -inf have no weight.  (float64 throughout: its
    // pipe takes a warp's operation in two cycles, and what integers and tables did instead took twice as long.)
    __device__ __forceinline__ double scaled(float x) const {
        const double y = (static_cast<double>(x) - static_cast<double>(top)) * c;
        const double magic = 6755399441055744.0;                      // 1.5 2^52: adding it rounds to an integer
        const double shifted = y + magic;
        const double p = exp2_taylor<12>(y - (shifted - magic));
        const int n = __double2loint(shifted) + kFraction;
        const double w = __hiloint2double(__double2hiint(p) + (n << 20), __double2loint(p));
        if (x == top) return static_cast<double>(1ull << kFraction);   // (infinite ones, too: y is not a number then)
        return y >= -static_cast<double>(kFraction) ? w : 0.0;         // (else `w` may be anything)
    }
    __device__ __forceinline__ static u64 rounded(double scaled) {
        const double shifted = scaled + 4503599627370496.0;            // 2^52: the integer is in the low bits
        return static_cast<u64>(__double_as_longlong(shifted)) & ((1ull << 52) - 1);
    }
    __device__ __forceinline__ u64 weight(float x) const { return rounded(scaled(x)); }
    // falls (or stays) as x grows
    template <int BINS>
    __device__ __forceinline__ int bin(float x) const {
        return x == top ? 0 : static_cast<int>(fminf((top - x) * (bins * (BINS - 1)), static_cast<float>(BINS - 1)));
    }
};

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_scan64(u64 v, int lane) {          // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
    }
    return v;
}

// The smallest key in [lo, hi] for which `holds` (false up to some key, true behind it; true at hi).  One warp.
template <typename F>
__device__ __forceinline__ unsigned first_key(unsigned lo, unsigned hi, int lane, F holds) {
    while (lo < hi) {
        const unsigned step = (hi - lo) / 32 + 1;
        const u64 at = static_cast<u64>(lo) + static_cast<u64>(step) * lane;
        const unsigned probe = at < hi ? static_cast<unsigned>(at) : hi;
        const unsigned yes = __ballot_sync(0xffffffffu, holds(probe));
        const int first = __ffs(yes) - 1;    // (lane 31's probe may be below hi: then none may hold)
        if (first < 0) {
            lo = static_cast<unsigned>(lo + static_cast<u64>(step) * 31) + 1;
        } else {
            const u64 end = static_cast<u64>(lo) + static_cast<u64>(step) * first;
            const unsigned next_hi = end < hi ? static_cast<unsigned>(end) : hi;
            lo = first > 0 ? static_cast<unsigned>(lo + static_cast<u64>(step) * (first - 1)) + 1 : lo;
            hi = next_hi;
        }
    }
    return lo;
}

// The keys of logits in [klo, khi] that fall into bin `bin` (counted from the maximum).  One warp.
template <int BINS>
__device__ __forceinline__ void keys_of_bin(const Heat& heat, int bin, int lane, unsigned& klo, unsigned& khi) {
    const unsigned lo = first_key(klo, khi, lane, [&](unsigned k) { return heat.template bin<BINS>(value_of(k)) <= bin; });
    if (bin > 0) khi = first_key(lo, khi, lane, [&](unsigned k) { return heat.template bin<BINS>(value_of(k)) < bin; }) - 1;
    klo = lo;
}

// The cut of an order at `target`: the last key of which some token has (mass of larger keys) <= target.
struct Cut {
    unsigned key;
    u64 above, mass;                         // of larger keys; of the logits equal to it
};

// MASS: weights; else every token counts 1.  The cut lies in keys [klo, khi]; `above` is the mass of larger ones; `binned`: they
// are one bin of the first histogram.
template <bool MASS, typename At>
__device__ Cut find_cut(cg::cluster_group& cluster, Shared& s, const Heat& heat, At at, int lo_i, int hi_i, unsigned klo,
                        unsigned khi, u64 above, bool binned, u64 target, int& level) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned ranks = cluster.num_blocks();
    for (int pass = binned ? 1 : 0;; ++pass, ++level) {
        u64* hist = s.hist[level & 1];
        for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
        if (tid == 0) s.cross_bin = kBins;
        __syncthreads();
        const int bits = 32 - __clz(khi - klo);
        const int shift = bits > 10 ? bits - 10 : 0;
        for (int i = lo_i + lane; i < hi_i; i += 32) {
            const float x = at(i);
            const unsigned key = key_of(x);
            if (key < klo || key > khi) continue;
            const int bin = pass == 0 ? kBins - 1 - heat.bin<kBins>(x) : static_cast<int>((key - klo) >> shift);
            const u64 w = MASS ? heat.weight(x) : 1ull;
            if (w) atomicAdd(hist + bin, w);
        }
        cluster.sync();
        // every CTA adds all of them up; thread t the bins 1023 - 2 t and 1022 - 2 t
        u64 m[2] = {0, 0};
        const int b0 = kBins - 1 - 2 * tid;
        for (unsigned r = 0; r < ranks; ++r) {
            const u64* other = cluster.map_shared_rank(hist, r);
            m[0] += other[b0];
            m[1] += other[b0 - 1];
        }
        const u64 incl = warp_scan64(m[0] + m[1], lane);
        if (lane == 31) s.scan[warp] = incl;
        __syncthreads();
        u64 before = above + incl - (m[0] + m[1]);
        for (int w = 0; w < warp; ++w) before += s.scan[w];
        const u64 a[2] = {before, before + m[0]};
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (m[j] && a[j] <= target) atomicMin(&s.cross_bin, b0 - j);
        __syncthreads();
        const int cross = s.cross_bin;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (b0 - j == cross) {
                s.cross_above = a[j];
                s.cross_mass = m[j];
            }
        if (pass == 0 && warp == 0) {
            // the keys whose logits fall into the bin
            unsigned lo = klo, hi = khi;
            keys_of_bin<kBins>(heat, kBins - 1 - cross, lane, lo, hi);
            if (lane == 0) {
                s.lo = lo;
                s.hi = hi;
            }
        }
        __syncthreads();
        above = s.cross_above;
        const u64 mass = s.cross_mass;
        if (pass == 0) {
            klo = s.lo;
            khi = s.hi;
        } else {
            const unsigned first = klo + (static_cast<unsigned>(cross) << shift);
            khi = min(khi, first + ((1u << shift) - 1u));
            klo = first;
        }
        __syncthreads();
        if (klo == khi) {
            ++level;
            return Cut{klo, above, mass};
        }
    }
}

// f(index, logit) for a warp's segment [lo_i, hi_i), 16 bytes of logits a lane at a time (not in the order of indices).
template <typename T, typename F>
__device__ __forceinline__ void each_logit(const T* seg, int n, int lane, F f) {
    constexpr int VEC = 16 / sizeof(T);
    const int whole = n / VEC;
    for (int i = lane; i < whole; i += 32) {
        const uint4 q = reinterpret_cast<const uint4*>(seg)[i];
        const T* v = reinterpret_cast<const T*>(&q);
#pragma unroll
        for (int e = 0; e < VEC; ++e) f(i * VEC + e, to_float(v[e]));
    }
    for (int i = whole * VEC + lane; i < n; i += 32) f(i, to_float(seg[i]));
}

// Inclusive scan over the block, in the order of threads.  Ends with all threads together.
__device__ __forceinline__ u64 block_scan64(u64 v, u64* scratch, u64& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 incl = warp_scan64(v, lane);
    __syncthreads();
    if (lane == 31) scratch[warp] = incl;
    __syncthreads();
    u64 before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const u64 x = scratch[w];
        if (w < warp) before += x;
        sum += x;
    }
    total = sum;
    return before + incl;
}

// `n` different numbers of v in descending order, by their ranks or, where they are many, in a network.  Zeros behind them up to a
// power of two.  Begins and ends with all threads together.
__device__ __forceinline__ void sort_descending(u64* v, int n) {
    const int tid = threadIdx.x;
    if (n <= kThreads / 2) {
        // 512 / size threads a number, neighbours in a warp (at most 32)
        int size = 16;
        while (size < n) size *= 2;
        const int each = kThreads / size, i = tid / each, part = tid % each;
        const u64 mine = i < n ? v[i] : 0ull;
        unsigned rank = 0;
        if (i < n)
            for (int j = part; j < n; j += each) rank += v[j] > mine ? 1u : 0u;
        for (int o = 1; o < each; o *= 2) rank += __shfl_xor_sync(0xffffffffu, rank, o);
        __syncthreads();
        if (i < n && part == 0) v[rank] = mine;
        __syncthreads();
        return;
    }
    int size = kThreads;
    while (size < n) size *= 2;
    for (int i = n + tid; i < size; i += kThreads) v[i] = 0ull;
    for (int run = 2; run <= size; run *= 2)
        for (int step = run / 2; step > 0; step /= 2) {
            __syncthreads();
            for (int t = tid; t < size / 2; t += kThreads) {
                const int i = 2 * t - (t & (step - 1)), j = i + step;
                const u64 a = v[i], b = v[j];
                if ((a < b) == ((i & run) == 0)) {
                    v[i] = b;
                    v[j] = a;
                }
            }
        }
    __syncthreads();
}

__device__ __forceinline__ u64 drawn_mass(float u, u64 z) {
    const u64 target = u > 0.f ? static_cast<u64>(static_cast<double>(u) * static_cast<double>(z)) : 0ull;
    return min(target, z - 1);
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
draw_kernel(const T* __restrict__ logits, long long stride, int V, int seg, Settings set, const float* __restrict__ uniform,
            int draws, int* __restrict__ out, float* __restrict__ prob) {
    extern __shared__ __align__(16) unsigned char slice_raw[];
    __shared__ __align__(16) Shared s;
    T* slice = reinterpret_cast<T*>(slice_raw);                // kWarps segments of `seg`
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned rank = cluster.block_rank(), ranks = cluster.num_blocks();
    const int row = blockIdx.x / ranks;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = (static_cast<int>(rank) * kWarps) * seg;       // the CTA's first token
    const int lo_i = min(first + warp * seg, V), hi_i = min(first + (warp + 1) * seg, V);
    const int mine_n = hi_i - lo_i;                            // logits of this warp's segment

    pdl_launch_dependents();
    if (tid == 0) {
        mbar_init(smem_u32(&s.loaded), 1);
        s.bin_count = 0;
        mbar_fence_init();
    }
    // (another CTA's shared memory may be written only once that CTA runs: all have said so in front of the first exchange, and
    // the answer arrives behind the copy)
    auto running = cluster.barrier_arrive();
    pdl_wait();
    const T* x_row = logits + row * stride + first;
    const int slice_n = max(min(first + kWarps * seg, V) - first, 0);
    const bool bulk = (reinterpret_cast<uintptr_t>(x_row) & 15) == 0;
    const int bulk_n = bulk ? slice_n / (16 / static_cast<int>(sizeof(T))) * (16 / static_cast<int>(sizeof(T))) : 0;
    __syncthreads();
    if (tid == 0 && bulk_n > 0) {
        const uint32_t bytes = static_cast<uint32_t>(bulk_n) * sizeof(T);
        mbar_expect_tx(smem_u32(&s.loaded), bytes);
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(smem_u32(slice)),
                     "l"(x_row), "r"(bytes), "r"(smem_u32(&s.loaded))
                     : "memory");
    }
    for (int i = bulk_n + tid; i < slice_n; i += kThreads) slice[i] = x_row[i];
    const float heat_in = set.temperature[row];
    const int k_in = set.top_k[row];
    const float p = set.top_p[row], least = set.min_p[row] > 0.f ? fminf(set.min_p[row], 1.0f) : 0.f;
    const int k = k_in > 0 && k_in < V ? k_in : 0;
    bool arrived = true;
    if (bulk_n > 0) arrived = mbar_wait(smem_u32(&s.loaded), 0);
    if (!arrived) atomicExch(&g_draw_error, 1);
    __syncthreads();
    // the first CTA's survivors: by value, their weights, and in the order of indices (in its slice's place, once it is done with that)
    u64* const order = reinterpret_cast<u64*>(slice_raw);
    u64* const weight_of = order + kListed;
    Token* const all_of = reinterpret_cast<Token*>(weight_of + kListed);
    auto at = [&](int i) { return logit_of(to_float(slice[i - first])); };
    const T* my_seg = slice + (lo_i - first);
    if (set.penalty) {
        // tokens of the history, each named once: x / penalty where x > 0, x * penalty elsewhere
        const float pen = set.penalty[row];
        if (pen != 1.0f)
            for (int h = set.hist_off[row] + tid; h < set.hist_off[row + 1]; h += kThreads) {
                const int i = set.hist_tok[h];
                if (i < first || i >= first + slice_n) continue;
                const float x = at(i);
                slice[i - first] = from_float<T>(x > 0.f ? x / pen : x * pen);
            }
        __syncthreads();
    }

    // ---- the maximum; and a key that at least k logits of the row reach, by the largest logits of warps or threads
    float mx = -INFINITY;
    each_logit(my_seg, mine_n, lane, [&](int, float x) { mx = fmaxf(mx, x); });      // (NaN counts as -inf)
    const unsigned mx_key = key_of(mx + 0.0f);
    const unsigned warp_top = __reduce_max_sync(0xffffffffu, mx_key);
    if (lane == 0) s.key[warp] = warp_top;
    unsigned floor_key = 0;
    const int r = (k + static_cast<int>(ranks) - 1) / static_cast<int>(ranks);
    __syncthreads();
    if (k > 0 && heat_in > 0.f) {
        if (r <= kWarps) {
            // (of the warps' maxima, where these are enough)
            const unsigned mine = s.key[lane & (kWarps - 1)];
            int larger = 0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) larger += s.key[w] > mine ? 1 : 0;
            floor_key = __reduce_min_sync(0xffffffffu, larger < r ? mine : 0xffffffffu);
        } else if (r <= kThreads) {
            for (int bit = 31; bit >= 16; --bit) {
                const unsigned next = floor_key | (1u << bit);
                if (__syncthreads_count(mx_key >= next) >= r) floor_key = next;
            }
        }
    }
    cluster.barrier_wait(std::move(running));                  // every CTA of the cluster has begun
    if (tid < static_cast<int>(ranks)) {
        unsigned best = 0;
        for (int w = 0; w < kWarps; ++w) best = max(best, s.key[w]);
        *cluster.map_shared_rank(&s.top_key[rank], tid) = best;
        *cluster.map_shared_rank(&s.floor_key[rank], tid) = floor_key;
    }
    cluster.sync();
    unsigned best = 0;
    floor_key = 0xffffffffu;
    for (unsigned c = 0; c < ranks; ++c) {
        best = max(best, s.top_key[c]);
        floor_key = min(floor_key, s.floor_key[c]);
    }
    const float top = value_of(best);
    const long long draw0 = static_cast<long long>(row) * draws;
    if (!(heat_in > 0.f) || top == -INFINITY) {
        // greedy: the lowest index of the maximum; a row in which every logit is -inf has no token to draw: token 0,
        // with probability 0
        int lowest = 0x7fffffff;
        each_logit(my_seg, mine_n, lane, [&](int i, float x) { if (x == top) lowest = min(lowest, lo_i + i); });
        lowest = static_cast<int>(__reduce_min_sync(0xffffffffu, static_cast<unsigned>(lowest)));
        if (lane == 0) s.at[warp] = lowest;
        __syncthreads();
        if (tid == 0) {
            unsigned l = 0x7fffffff;
            for (int w = 0; w < kWarps; ++w) l = min(l, s.at[w]);
            *cluster.map_shared_rank(&s.top_at[rank], 0) = l;
        }
        cluster.sync();
        if (rank == 0) {
            unsigned l = 0x7fffffff;
            for (unsigned c = 0; c < ranks; ++c) l = min(l, s.top_at[c]);
            for (int j = tid; j < draws; j += kThreads) {
                out[draw0 + j] = top == -INFINITY ? 0 : static_cast<int>(l);
                if (prob) prob[draw0 + j] = top == -INFINITY ? 0.f : 1.f;
            }
        }
        return;                              // (nobody reads another CTA's memory any more)
    }
    Heat heat;
    heat.top = top;
    heat.c = 1.4426950408889634074 / static_cast<double>(heat_in);
    heat.bins = 1.0f / (30.5f * heat_in);
    const double bound = least > 0.f ? static_cast<double>(least) * static_cast<double>(1ull << kFraction) : 0.0;

    // the sum of `mine` over all warps of the cluster
    auto cluster_sum = [&](u64 mine, u64* exchange) {
        mine = warp_sum64(mine);
        if (lane == 0) s.warp_sum[warp] = mine;
        __syncthreads();
        if (tid < static_cast<int>(ranks)) {
            u64 sum = 0;
            for (int w = 0; w < kWarps; ++w) sum += s.warp_sum[w];
            *cluster.map_shared_rank(&exchange[rank], tid) = sum;
        }
        cluster.sync();
        u64 z = 0;
        for (unsigned c = 0; c < ranks; ++c) z += exchange[c];
        return z;
    };
    bool cut_known = false;                  // top-p's, in s.cut_key and s.tie_cut
    int bin_count = 0;                       // tokens of its bin in this CTA, in s.bin_list
    const bool filtered = k > 0 || p < 1.0f || bound > 0.0;
    // ---- top-p over the whole row: its mass, and the bin of its cut
    u64 whole = 0, bin_above = 0, target = 0;
    u64 above_here = 0;                      // of that, this thread's share of what its CTA has above the bin
    unsigned bin_lo = 0, bin_hi = 0;
    if (k == 0 && p < 1.0f) {
        // exact sums by 32-bit additions: a weight in three pieces of 15 bits (fewer than 2^17 of them a bin and CTA), most of
        // which are nothing
        for (int i = tid; i < 3 * kMassBins; i += kThreads) (&s.pieces[0][0])[i] = 0;
        if (tid == 0) s.cross_bin = -1;
        __syncthreads();
        auto add_to_bin = [&](float x, unsigned times) {
            const u64 w = heat.weight(x);    // (NaN: none)
            if (!w) return;
            const int bin = heat.bin<kMassBins>(x);
            const unsigned a = static_cast<unsigned>(w) & 32767u, b = static_cast<unsigned>(w >> 15) & 32767u, c = static_cast<unsigned>(w >> 30);
            if (a) atomicAdd(&s.pieces[0][bin], a * times);
            if (b) atomicAdd(&s.pieces[1][bin], b * times);
            if (c) atomicAdd(&s.pieces[2][bin], c * times);
        };
        bool counted = false;
        if constexpr (sizeof(T) == 2) {
            // Logits of 16 bits have few values: those of sixteen exponents are counted (two counters of 16 bits a word), and a
            // weight is computed once a value; others, next to zero or far from it, are weighed one by one.
            __shared__ unsigned counts[kCounted / 2];
            counted = slice_n >= 4 * kCounted && slice_n < 65536;
            if (counted) {
                for (int i = tid; i < kCounted / 2; i += kThreads) counts[i] = 0;
                __syncthreads();
                each_logit(my_seg, mine_n, lane, [&](int, float x) {
                    const unsigned bits = __float_as_uint(x), at = ((bits >> 16) & 0x7fffu) - kCountedFrom;
                    if (at < kCounted / 2) {
                        // (a value and its negative share a word)
                        atomicAdd(&counts[at], (bits >> 31) ? 65536u : 1u);
                    } else {
                        add_to_bin(x, 1u);
                    }
                });
                __syncthreads();
                for (int i = tid; i < kCounted / 2; i += kThreads) {
                    const unsigned n = counts[i];
                    const float x = __uint_as_float((i + kCountedFrom) << 16);
                    if (n & 0xffffu) add_to_bin(x, n & 0xffffu);
                    if (n >> 16) add_to_bin(-x, n >> 16);
                }
            }
        }
        if (!counted) each_logit(my_seg, mine_n, lane, [&](int, float x) { add_to_bin(x, 1u); });
        cluster.sync();
        // a CTA adds its share of the bins up, then all of them learn each share's mass, then where the cut lies
        constexpr int EACH = kMassBins / kThreads;                   // bins of a thread at most
        const int share = kMassBins / static_cast<int>(ranks);       // (128 to 2,048)
        const int each = max(share / kThreads, 1);
        u64 m[EACH] = {}, sum_m = 0;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int bin = each * tid + e;
            if (e < each && bin < share)
                for (unsigned c = 0; c < ranks; ++c) {
                    const unsigned* other = cluster.map_shared_rank(&s.pieces[0][0], c) + rank * share + bin;
#pragma unroll
                    for (int q = 0; q < 3; ++q) m[e] += static_cast<u64>(other[q * kMassBins]) << (15 * q);
                }
            sum_m += m[e];
        }
        u64 here;
        const u64 incl = block_scan64(sum_m, s.scan, here);
        if (tid < static_cast<int>(ranks)) *cluster.map_shared_rank(&s.total[rank], tid) = here;
        cluster.sync();
        u64 in_front = 0, of_the_cut = 0;
        for (unsigned c = 0; c < ranks; ++c) whole += s.total[c];
        target = static_cast<u64>(static_cast<double>(fmaxf(p, 0.f)) * static_cast<double>(whole));
        int owner = -1;                      // the last share that has some mass and no more than the target in front of it
        for (unsigned c = 0; c < ranks; ++c) {
            if (s.total[c] && in_front <= target) {
                owner = static_cast<int>(c);
                of_the_cut = in_front;
            }
            in_front += s.total[c];
        }
        if (owner == static_cast<int>(rank)) {
            u64 in_front_of = of_the_cut + incl - sum_m;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                if (m[e] && in_front_of <= target) atomicMax(&s.cross_bin, each * tid + e);
                in_front_of += m[e];
            }
            __syncthreads();
            const int cross = s.cross_bin;   // (>= 0: the share's first bin with mass qualifies)
            in_front_of = of_the_cut + incl - sum_m;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                if (e < each && each * tid + e == cross) s.cross_above = in_front_of;
                in_front_of += m[e];
            }
            if (warp == 0) {
                unsigned lo = 0, hi = best;
                keys_of_bin<kMassBins>(heat, static_cast<int>(rank) * share + cross, lane, lo, hi);
                if (lane == 0) {
                    s.lo = lo;
                    s.hi = hi;
                }
            }
            __syncthreads();
            const unsigned found_lo = s.lo, found_hi = s.hi;
            const u64 found = s.cross_above;
            __syncthreads();
            if (tid < static_cast<int>(ranks)) {
                *cluster.map_shared_rank(&s.lo, tid) = found_lo;
                *cluster.map_shared_rank(&s.hi, tid) = found_hi;
                *cluster.map_shared_rank(&s.cross_above, tid) = found;
                *cluster.map_shared_rank(&s.cross_bin, tid) = static_cast<int>(rank) * share + cross;
            }
        }
        cluster.sync();                      // (nobody reads another CTA's pieces any more)
        for (int bin = tid; bin < s.cross_bin; bin += kThreads)
#pragma unroll
            for (int q = 0; q < 3; ++q) above_here += static_cast<u64>(s.pieces[q][bin]) << (15 * q);
        __syncthreads();
        bin_lo = s.lo;
        bin_hi = s.hi == 0x7fffffffu ? s.hi - 1 : s.hi;      // (the key of -0, which no logit has: as a float it equals 0)
        bin_above = s.cross_above;
    }
    if (filtered) {
        // ---- what can be kept at all: keys from floor_key on
        if (k == 0) floor_key = bin_lo;      // (0 without top-p)
        if (bound > 0.0 && (k == 0 || p >= 1.0f)) {
            if (warp == 0) {
                const unsigned lowest = first_key(key_of(-INFINITY), best, lane, [&](unsigned q) { return heat.scaled(value_of(q)) >= bound; });
                if (lane == 0) s.key[0] = lowest;
            }
            __syncthreads();
            floor_key = max(floor_key, s.key[0]);
            __syncthreads();
        }
        // counted and listed: the survivors, in the order of indices, and where top-p's bin is known its tokens
        const unsigned bin_top = k == 0 && p < 1.0f ? bin_hi : 0u;
        unsigned mine = 0;
        const bool take_all = floor_key <= key_of(-INFINITY);        // (NaN, too)
        const float floor_x = value_of(max(floor_key, key_of(-INFINITY)));
        const float bin_lo_x = bin_top ? value_of(max(bin_lo, key_of(-INFINITY))) : INFINITY, bin_hi_x = bin_top ? value_of(bin_hi) : -INFINITY;
        auto in_all = [&](float x) { return x >= floor_x || take_all; };
        auto in_bin = [&](float x) { return x >= bin_lo_x && x <= bin_hi_x; };      // (not NaN: it has no weight)
        each_logit(my_seg, mine_n, lane, [&](int i, float x) {
            mine += in_all(x) ? 1u : 0u;
            if (in_bin(x)) {
                const unsigned slot = atomicAdd(&s.bin_count, 1u);
                if (slot < kBinListed) s.bin_list[slot] = Token{key_of(logit_of(x)), lo_i + i};
            }
        });
        mine = __reduce_add_sync(0xffffffffu, mine);
        if (lane == 0) s.key[warp] = mine;
        __syncthreads();
        unsigned before = 0;
        uint2 here = make_uint2(0, s.bin_count);                     // (survivors, tokens of the bin)
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += s.key[w];
            here.x += s.key[w];
        }
        if (here.x <= kListed && mine) {
            for (int i0 = 0; i0 < mine_n; i0 += 128) {
                float x[4];
                bool in = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = i0 + 32 * e + lane;
                    x[e] = i < mine_n ? to_float(my_seg[i]) : 0.f;
                    in = in || (i < mine_n && in_all(x[e]));
                }
                if (!__any_sync(0xffffffffu, in)) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = i0 + 32 * e + lane;
                    const bool hit = i < mine_n && in_all(x[e]);
                    const unsigned hits = __ballot_sync(0xffffffffu, hit);
                    if (hit) s.list[before + __popc(hits & ((1u << lane) - 1))] = Token{key_of(logit_of(x[e])), lo_i + i};
                    before += __popc(hits);
                }
            }
        }
        if (tid < static_cast<int>(ranks)) *cluster.map_shared_rank(&s.listed[rank], tid) = here;
        cluster.sync();
        unsigned n = 0, n_bin = 0;
        for (unsigned c = 0; c < ranks; ++c) {
            n += s.listed[c].x;              // (fewer than 2^20 together)
            n_bin += s.listed[c].y;
        }
        // the first CTA's share of a list in all CTAs: `take` (place, token)
        auto gather = [&](bool bins, unsigned count, auto take) {
            for (unsigned i = tid; rank == 0 && i < count; i += kThreads) {
                unsigned c = 0, from = 0;
                for (unsigned end = bins ? s.listed[0].y : s.listed[0].x; i >= end; end += bins ? s.listed[c].y : s.listed[c].x) {
                    from = end;
                    ++c;
                }
                const Token* other = bins ? cluster.map_shared_rank(s.bin_list, c) : cluster.map_shared_rank(s.list, c);
                take(i, other[i - from]);
            }
        };
        if (n > kListed && bin_top && n_bin <= kBinListed) {
            // ---- the first CTA finds top-p's cut among the tokens of its bin
            gather(true, n_bin, [&](unsigned i, Token t) { s.bin_order[i] = (static_cast<u64>(t.key) << 32) | (0xffffffffu - t.at); });
            if (rank == 0) {
                __syncthreads();
                sort_descending(s.bin_order, static_cast<int>(n_bin));
                u64 w[2], sum;
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    w[e] = 2 * tid + e < static_cast<int>(n_bin) ? heat.weight(value_of(static_cast<unsigned>(s.bin_order[2 * tid + e] >> 32))) : 0ull;
                const u64 incl = block_scan64(w[0] + w[1], s.scan, sum);
                const int kept = __syncthreads_count(w[0] && bin_above + incl - w[0] - w[1] <= target) +
                                 __syncthreads_count(w[1] && bin_above + incl - w[1] <= target);
                if (tid < static_cast<int>(ranks)) {
                    const u64 last = s.bin_order[max(kept, 1) - 1];
                    *cluster.map_shared_rank(&s.cut_key, tid) = static_cast<unsigned>(last >> 32);
                    *cluster.map_shared_rank(&s.tie_cut, tid) = static_cast<int>(0xffffffffu - static_cast<unsigned>(last));
                }
            }
            cluster.sync();
            cut_known = true;
            bin_count = static_cast<int>(here.y);
        }
        if (n <= kListed) {
            // ---- the first CTA takes it from here
            gather(false, n, [&](unsigned i, Token t) { all_of[i] = t; });
            cluster.sync();                  // (the others' lists have been read)
            if (rank != 0) return;
            const int count = static_cast<int>(n);
            for (int i = tid; i < count; i += kThreads) order[i] = (static_cast<u64>(all_of[i].key) << 32) | (0xffffffffu - i);
            __syncthreads();
            sort_descending(order, count);
            // weights by value, kEach a thread; what top-k leaves
            constexpr int kEach = kListed / kThreads;
            const int nk = k > 0 ? min(k, count) : count;
            double scaled[kEach];
            u64 w[kEach], sum_w = 0;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int i = kEach * tid + e;
                scaled[e] = i < nk ? heat.scaled(value_of(static_cast<unsigned>(order[i] >> 32))) : -1.0;
                w[e] = i < nk ? Heat::rounded(scaled[e]) : 0ull;
                sum_w += w[e];
            }
            u64 sum;
            u64 front = block_scan64(sum_w, s.scan, sum) - sum_w;
            const u64 z_top = k > 0 ? sum : whole;
            target = static_cast<u64>(static_cast<double>(fmaxf(p, 0.f)) * static_cast<double>(z_top));
            for (int i = tid; i < count; i += kThreads) weight_of[i] = 0;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                if (scaled[e] >= bound && (!(p < 1.0f) || front <= target))
                    weight_of[0xffffffffu - static_cast<unsigned>(order[kEach * tid + e])] = w[e];
                front += w[e];
            }
            __syncthreads();
            // cumulated in the order of indices
            u64 z;
            sum_w = 0;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int i = kEach * tid + e;
                w[e] = i < count ? weight_of[i] : 0ull;
                sum_w += w[e];
            }
            front = block_scan64(sum_w, s.scan, z) - sum_w;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                front += w[e];
                if (kEach * tid + e < count) weight_of[kEach * tid + e] = front;
            }
            __syncthreads();
            for (int j = tid; j < draws; j += kThreads) {
                const u64 goal = drawn_mass(uniform[draw0 + j], z);
                int lo = 0, hi = count - 1;
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (weight_of[mid] > goal) hi = mid;
                    else lo = mid + 1;
                }
                out[draw0 + j] = all_of[lo].at;
                if (prob) prob[draw0 + j] = static_cast<float>(heat.scaled(value_of(all_of[lo].key)) / static_cast<double>(z));
            }
            return;
        }
    }

    // ---- no filter, or too many survivors for one CTA: what is kept is keys above cut_key, and logits equal to it up to
    // index tie_cut
    unsigned cut_key = 0;
    int tie_cut = 0x7fffffff, level = 0;
    u64 ties = 0, ties_kept = 0;
    if (k > 0) {
        const Cut c = find_cut<false>(cluster, s, heat, at, lo_i, hi_i, 0u, best, 0ull, false, static_cast<u64>(k - 1), level);
        cut_key = c.key;
        ties = c.mass;
        ties_kept = min(ties, static_cast<u64>(k) - c.above);
    }
    if (cut_known) {
        cut_key = s.cut_key;
        tie_cut = s.tie_cut;
    } else if (p < 1.0f) {
        u64 z = whole;
        if (k > 0) {
            u64 mine = 0;
            for (int i = lo_i + lane; i < hi_i; i += 32) {
                const float x = at(i);
                const unsigned key = key_of(x);
                if (key > cut_key || (key == cut_key && ties == ties_kept)) mine += heat.weight(x);
            }
            z = cluster_sum(mine, s.mass);
            if (ties != ties_kept) z += ties_kept * heat.weight(value_of(cut_key));
        }
        target = static_cast<u64>(static_cast<double>(fmaxf(p, 0.f)) * static_cast<double>(z));
        const Cut c = k > 0 ? find_cut<true>(cluster, s, heat, at, lo_i, hi_i, cut_key, best, 0ull, false, target, level)
                            : find_cut<true>(cluster, s, heat, at, lo_i, hi_i, bin_lo, bin_hi, bin_above, true, target, level);
        const u64 w = heat.weight(value_of(c.key));
        const u64 there = c.key == cut_key && ties ? ties_kept : c.mass / w;    // tokens of that key which top-k left
        const u64 all = c.key == cut_key && ties ? ties : there;
        cut_key = c.key;
        ties = all;
        ties_kept = min(there, (target - c.above) / w + 1);
    }
    if (bound > 0.0) {
        // the smallest key whose weight is min-p of the largest
        if (warp == 0) {
            const unsigned lowest = first_key(key_of(-INFINITY), best, lane, [&](unsigned q) { return heat.scaled(value_of(q)) >= bound; });
            if (lane == 0) s.lo = lowest;
        }
        __syncthreads();
        if (s.lo > cut_key) {
            cut_known = false;
            cut_key = s.lo;
            ties = ties_kept = 0;
            tie_cut = 0x7fffffff;
        }
    }
    if (ties_kept < ties) {
        // the index of the last of the equal logits that are kept
        unsigned mine = 0;
        for (int i = lo_i + lane; i < hi_i; i += 32) mine += key_of(at(i)) == cut_key ? 1u : 0u;
        mine = __reduce_add_sync(0xffffffffu, mine);
        __syncthreads();
        if (lane == 0) s.key[warp] = mine;
        __syncthreads();
        if (tid < static_cast<int>(ranks)) {
            unsigned sum = 0;
            for (int w = 0; w < kWarps; ++w) sum += s.key[w];
            *cluster.map_shared_rank(&s.ties[rank], tid) = sum;
        }
        cluster.sync();
        u64 before = 0;
        for (unsigned c = 0; c < rank; ++c) before += s.ties[c];
        for (int w = 0; w < warp; ++w) before += s.key[w];
        // (tie_cut is this warp's own: all of its tokens in front of the last kept tie, behind it none)
        if (before >= ties_kept) {
            tie_cut = -1;
        } else if (before + mine > ties_kept) {
            u64 left = ties_kept - before;
            for (int base = lo_i; base < hi_i; base += 32) {
                const unsigned hit = __ballot_sync(0xffffffffu, base + lane < hi_i && key_of(at(min(base + lane, hi_i - 1))) == cut_key);
                const unsigned n = __popc(hit);
                if (n >= left) {
                    tie_cut = base + __fns(hit, 0, static_cast<int>(left));
                    break;
                }
                left -= n;
            }
        }
    }
    // (as floats: key 0 is below all of them, and NaN, which has no weight, is never larger)
    const bool cut_none = cut_key < key_of(-INFINITY);
    const float cut_x = cut_none ? -INFINITY : value_of(cut_key);
    auto kept_weight = [&](int i, float x) -> u64 {
        return x > cut_x || (x == cut_x && i <= tie_cut) ? heat.weight(x) : 0ull;
    };

    // Where the cut lies in a bin whose tokens are listed, the bins above it say what this CTA keeps: the row's mass is
    // known, and only a CTA on which a number falls looks for its token.
    u64 z = 0, from = 0;
    if (cut_known) {
        u64 mine = above_here;
        for (int i = tid; i < bin_count; i += kThreads) {
            const Token token = s.bin_list[i];
            mine += kept_weight(token.at, value_of(token.key));
        }
        z = cluster_sum(mine, s.total);
        for (unsigned c = 0; c < rank; ++c) from += s.total[c];
        bool some = false;
        for (int j = tid; j < draws; j += kThreads) {
            const u64 goal = drawn_mass(uniform[draw0 + j], z);
            some = some || (goal >= from && goal < from + s.total[rank]);
        }
        if (!__syncthreads_or(some)) return;
    }
    // ---- masses: a lane's are those of a contiguous block of its warp's segment (an odd number of tokens: no two lanes
    // of a warp in one bank)
    const int block_n = ((seg + 31) / 32) | 1;
    const int b0 = min(lane * block_n, mine_n), b1 = min(b0 + block_n, mine_n);
    u64 mine = 0;
    for (int i = b0; i < b1; ++i) mine += kept_weight(lo_i + i, to_float(my_seg[i]));
    __syncthreads();                         // (warp_sum may still be read)
    if (cut_known) {
        const u64 sum = warp_sum64(mine);
        if (lane == 0) s.warp_sum[warp] = sum;
        __syncthreads();
    } else {
        z = cluster_sum(mine, s.total);
        for (unsigned c = 0; c < rank; ++c) from += s.total[c];
    }
    for (int w = 0; w < warp; ++w) from += s.warp_sum[w];
    from += warp_scan64(mine, lane) - mine;  // what lies in front of this lane's block
    // ---- the draws: each is taken by the warp on whose segment its number falls
    for (int j = 0; j < draws; ++j) {
        const u64 goal = drawn_mass(uniform[draw0 + j], z);
        const unsigned owner = __ballot_sync(0xffffffffu, goal >= from && goal < from + mine);
        if (!owner) continue;
        const int l = __ffs(owner) - 1;
        u64 sum = __shfl_sync(0xffffffffu, from, l);
        const int first_of = l * block_n, end_of = min(first_of + block_n, mine_n);
        for (int base = first_of; base < end_of; base += 32) {
            const int i = base + lane;
            const u64 w = i < end_of ? kept_weight(lo_i + i, to_float(my_seg[i])) : 0ull;
            const u64 incl = warp_scan64(w, lane) + sum;
            const unsigned over = __ballot_sync(0xffffffffu, incl > goal);
            if (over) {
                if (lane == __ffs(over) - 1) {
                    out[draw0 + j] = lo_i + i;
                    if (prob) prob[draw0 + j] = static_cast<float>(heat.scaled(at(lo_i + i)) / static_cast<double>(z));
                }
                break;
            }
            sum = __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    // (nobody reads another CTA's memory behind the last sum: all may leave)
}

// Tokens of a row, at most: the slices of the largest cluster, and sums of weights below 2^64.
template <typename T>
constexpr int most_tokens() {
    return std::min(kMaxCluster * kMostSlice / static_cast<int>(sizeof(T)), (1 << 20) - 1);
}

template <typename T>
int launch_draw(const void* logits, long long stride, int rows, int V, const Settings& set, const float* uniform, int draws,
                int* out, float* prob, cudaStream_t stream) {
    int ranks = 1;
    const auto bytes_of = [&](int n) { return static_cast<long long>(V) / n * static_cast<long long>(sizeof(T)); };
    // (16 CTAs a row while the rows' clusters find room beside each other.  152,064 float32 logits, 16 CTAs and 8: without filters 1 row
    // 9.2 us and 13.3, 8 rows 13.1 and 14.8, 12 rows 13.2 and 19.1, 16 rows 19.4 and 20.1, 24 rows 24.3 and 20.3; with top-p alone 31 and 42,
    // 41 and 46, 44 and 55, 59 and 54, 71 and 57; with top-k 50 11.3 and 12.8, 15.6 and 14.0, 14.9 and 15.7, 20.6 and 16.5, 22.7 and 17.2;
    // bfloat16 the same within a microsecond but for top-p, 12 rows 46.1 and 44.8.  32,000 logits take eight in any case.)
    while (ranks < (rows <= 12 ? kMaxCluster : 8) && V > ranks * 4096 && !(rows * ranks >= 256 && bytes_of(ranks) <= 78 * 1024)) ranks *= 2;
    const auto segment = [&](int n) { return ((V + n * kWarps - 1) / (n * kWarps) + 7) / 8 * 8; };
    while (ranks < kMaxCluster && static_cast<long long>(segment(ranks)) * kWarps * sizeof(T) > kMostSlice) ranks *= 2;
    const int seg = segment(ranks);
    const long long bytes = std::max(static_cast<long long>(seg) * kWarps * static_cast<long long>(sizeof(T)), 24ll * kListed);
    if (V > most_tokens<T>() || bytes > kMostSlice || static_cast<long long>(rows) * ranks > 0x7fffffffll) return SOMI_ERR_UNSUPPORTED;
    allow_smem<draw_kernel<T>>(kMostSlice);
    if (ranks > 8 && cudaFuncSetAttribute(draw_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
        return SOMI_ERR_UNSUPPORTED;
    return launch_pdl_cluster(draw_kernel<T>, dim3(static_cast<unsigned>(rows) * ranks), dim3(kThreads), static_cast<size_t>(bytes),
                              static_cast<unsigned>(ranks), stream, static_cast<const T*>(logits), stride, V, seg, set, uniform,
                              draws, out, prob);
}

}  // namespace draw
}  // namespace somi

using namespace somi;

SOMI_API int somi_draw_error() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, draw::g_draw_error, sizeof(int)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(draw::g_draw_error, &zero, sizeof(int));
    return v;
}

// The largest vocabulary of a type, 0 where it is not taken.
SOMI_API int somi_draw_max_vocabulary(int dtype) {
    return dtype == SOMI_F32 ? draw::most_tokens<float>() : dtype == SOMI_BF16 ? draw::most_tokens<__nv_bfloat16>() : 0;
}

// logits [rows, V] (rows `stride` elements apart), uniform, out and prob (or null) [rows, draws]; temperature, top_k,
// top_p, min_p [rows]; penalty [rows], hist_off [rows + 1] and hist_tok, or all null (float32 logits only).
SOMI_API int somi_draw(const void* logits, int dtype, long long stride, int rows, int V, const float* uniform, int draws,
                       const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                       const float* penalty, const int* hist_off, const int* hist_tok, int* out, float* prob,
                       cudaStream_t stream) {
    if (rows <= 0 || draws <= 0) return 0;
    if (V <= 0 || (penalty && (dtype != SOMI_F32 || !hist_off || !hist_tok))) return SOMI_ERR_UNSUPPORTED;
    const draw::Settings set{temperature, top_p, min_p, penalty, top_k, hist_off, hist_tok};
    if (dtype == SOMI_F32) return draw::launch_draw<float>(logits, stride, rows, V, set, uniform, draws, out, prob, stream);
    if (dtype == SOMI_BF16) return draw::launch_draw<__nv_bfloat16>(logits, stride, rows, V, set, uniform, draws, out, prob, stream);
    return SOMI_ERR_UNSUPPORTED;
}
