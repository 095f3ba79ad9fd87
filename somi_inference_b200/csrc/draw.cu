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
// polynomial, |r| <= 1/2, relative error 2e-16) and held as an integer multiple of 2^-44, and sums of integers
// are exact.  (Fewer than 2^20 weights of at most 2^44 stay below 2^64.)  So the result is the same bits
// whatever the launch looks like, and differs from real arithmetic only where a border lies within
// about 1e-11 of the number.
//
// A cluster of CTAs shares a row; each holds its slice in shared memory, read from HBM once.  A warp owns a
// contiguous segment of it.  All three cuts keep a beginning of one order, so what is kept is a key (the
// order-preserving integer image of a float), and an index up to which logits equal to it are kept.  The key
// is found by histograms that the cluster's CTAs add up: first over the logits' distance from
// the maximum (1,024 bins over the 30.5 temperatures in which weights do not vanish, so that a bin holds few
// tokens), then over the keys that lie in the bin of the cut, until a bin is one key.
#include <cooperative_groups.h>

#include "common.cuh"

namespace somi {
namespace draw {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 1024, kMaxCluster = 16;
constexpr int kFraction = 44;                // a weight is an integer multiple of 2^-44
typedef unsigned long long u64;

struct Settings {
    const float *temperature, *top_p, *min_p, *penalty;
    const int *top_k, *hist_off, *hist_tok;
};

struct Shared {
    u64 hist[2][kBins];                      // (read by the other CTAs of the cluster)
    u64 scan[kWarps];
    u64 warp_sum[kWarps];
    u64 total[kMaxCluster], mass[kMaxCluster];   // written by the other CTAs, one exchange each
    unsigned top_key[kMaxCluster], top_at[kMaxCluster], ties[kMaxCluster];
    unsigned key[kWarps], at[kWarps];
    u64 cross_above, cross_mass;
    int cross_bin;
    unsigned lo, hi;
    int tie_cut;
};

__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
// A logit: NaN counts as -inf, -0 as 0 (equal values must have equal keys).
__device__ __forceinline__ float logit_of(float x) { return x == x ? x + 0.0f : -INFINITY; }

// 2^r = 1 + r ln 2 (1 + r ln 2 / 2 (1 + r ln 2 / 3 (...))), to the N-th power of r
template <int N, int K = 0>
__device__ __forceinline__ double exp2_taylor(double r) {
    if constexpr (K == N) return 1.0;
    else return fma(exp2_taylor<N, K + 1>(r), r * (0.69314718055994530942 / (K + 1)), 1.0);
}

// A row's maximum and temperature: what a weight depends on.
struct Heat {
    float top;
    double c;                                // log2(e) / T
    float bins;                              // bins per unit of distance from the maximum

    // w 2^44 before it is rounded to an integer; 0 where w < 2^-44
    __device__ __forceinline__ double scaled(float x) const {
        if (x == top) return static_cast<double>(1ull << kFraction);
        const double y = (static_cast<double>(x) - static_cast<double>(top)) * c;
        if (!(y >= -static_cast<double>(kFraction))) return 0.0;       // (-inf, and inf - inf, too)
        const double magic = 6755399441055744.0;                      // 1.5 2^52: adding it rounds to an integer
        const double shifted = y + magic;
        const double r = y - (shifted - magic);
        const int n = static_cast<int>(__double_as_longlong(shifted));  // (the low bits)
        const double p = exp2_taylor<13>(r);
        return __longlong_as_double(__double_as_longlong(p) + (static_cast<long long>(n + kFraction) << 52));
    }
    __device__ __forceinline__ u64 weight(float x) const {
        const double shifted = scaled(x) + 4503599627370496.0;         // 2^52: the integer is in the low bits
        return static_cast<u64>(__double_as_longlong(shifted)) & ((1ull << 52) - 1);
    }
    // falls (or stays) as x grows
    __device__ __forceinline__ int bin(float x) const {
        return x == top ? 0 : static_cast<int>(fminf((top - x) * bins, static_cast<float>(kBins - 1)));
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

// The cut of an order at `target`: the last key of which some token has (mass of larger keys) <= target.
struct Cut {
    unsigned key;
    u64 above, mass;                         // of larger keys; of the logits equal to it
};

// MASS: weights; else every token counts 1.  Tokens with keys below `floor_key` are left out.
template <bool MASS, typename At>
__device__ Cut find_cut(cg::cluster_group& cluster, Shared& s, const Heat& heat, At at, int lo_i, int hi_i, unsigned floor_key,
                        u64 target, int& level) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned ranks = cluster.num_blocks();
    unsigned klo = floor_key, khi = key_of(heat.top);
    u64 above = 0;
    for (int pass = 0;; ++pass, ++level) {
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
            const int bin = pass == 0 ? kBins - 1 - heat.bin(x) : static_cast<int>((key - klo) >> shift);
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
            const int bin = kBins - 1 - cross;
            const unsigned lo = first_key(klo, khi, lane, [&](unsigned k) { return heat.bin(value_of(k)) <= bin; });
            const unsigned hi = bin == 0 ? khi : first_key(lo, khi, lane, [&](unsigned k) { return heat.bin(value_of(k)) < bin; }) - 1;
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

template <typename T>
__global__ void __launch_bounds__(kThreads)
draw_kernel(const T* __restrict__ logits, long long stride, int V, int seg, Settings set, const float* __restrict__ uniform,
            int draws, int* __restrict__ out, float* __restrict__ prob) {
    extern __shared__ __align__(16) unsigned char slice_raw[];
    __shared__ Shared s;
    T* slice = reinterpret_cast<T*>(slice_raw);                // kWarps segments of `seg`
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned rank = cluster.block_rank(), ranks = cluster.num_blocks();
    const int row = blockIdx.x / ranks;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = (static_cast<int>(rank) * kWarps) * seg;       // the CTA's first token
    const int lo_i = min(first + warp * seg, V), hi_i = min(first + (warp + 1) * seg, V);

    pdl_launch_dependents();
    pdl_wait();
    const T* x_row = logits + row * stride;
    for (int i = lo_i + lane; i < hi_i; i += 32) slice[i - first] = x_row[i];
    const float heat_in = set.temperature[row];
    auto at = [&](int i) { return logit_of(to_float(slice[i - first])); };
    if (set.penalty) {
        // tokens of the history, each named once: x / penalty where x > 0, x * penalty elsewhere
        const float pen = set.penalty[row];
        __syncthreads();
        if (pen != 1.0f)
            for (int h = set.hist_off[row] + tid; h < set.hist_off[row + 1]; h += kThreads) {
                const int i = set.hist_tok[h];
                if (i < first || i >= min(first + kWarps * seg, V)) continue;
                const float x = at(i);
                slice[i - first] = from_float<T>(x > 0.f ? x / pen : x * pen);
            }
        __syncthreads();
    }

    // ---- the maximum, and the lowest index that has it
    unsigned best = 0, best_at = 0x7fffffff;
    __syncwarp();
    for (int i = lo_i + lane; i < hi_i; i += 32) {
        const unsigned k = key_of(at(i));
        if (k > best) {
            best = k;
            best_at = i;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned k = __shfl_xor_sync(0xffffffffu, best, o), j = __shfl_xor_sync(0xffffffffu, best_at, o);
        if (k > best || (k == best && j < best_at)) {
            best = k;
            best_at = j;
        }
    }
    if (lane == 0) {
        s.key[warp] = best;
        s.at[warp] = best_at;
    }
    __syncthreads();
    if (tid < static_cast<int>(ranks)) {
        for (int w = 0; w < kWarps; ++w)
            if (w == 0 || s.key[w] > best || (s.key[w] == best && s.at[w] < best_at)) {
                best = s.key[w];
                best_at = s.at[w];
            }
        *cluster.map_shared_rank(&s.top_key[rank], tid) = best;
        *cluster.map_shared_rank(&s.top_at[rank], tid) = best_at;
    }
    cluster.sync();
    best = 0;
    for (unsigned r = 0; r < ranks; ++r)
        if (s.top_key[r] > best) {
            best = s.top_key[r];
            best_at = s.top_at[r];
        }
    const float top = value_of(best);
    const long long draw0 = static_cast<long long>(row) * draws;
    if (!(heat_in > 0.f) || top == -INFINITY) {
        // greedy; a row in which every logit is -inf has no token to draw: token 0, with probability 0
        if (rank == 0)
            for (int j = tid; j < draws; j += kThreads) {
                out[draw0 + j] = top == -INFINITY ? 0 : static_cast<int>(best_at);
                if (prob) prob[draw0 + j] = top == -INFINITY ? 0.f : 1.f;
            }
        cluster.sync();
        return;
    }
    Heat heat;
    heat.top = top;
    heat.c = 1.4426950408889634074 / static_cast<double>(heat_in);
    heat.bins = static_cast<float>(kBins - 1) / (30.5f * heat_in);

    // ---- what is kept: keys above cut_key, and logits equal to it up to index tie_cut
    unsigned cut_key = 0;
    int tie_cut = 0x7fffffff, level = 0;
    u64 ties = 0, ties_kept = 0;
    const int k = set.top_k[row];
    if (k > 0 && k < V) {
        const Cut c = find_cut<false>(cluster, s, heat, at, lo_i, hi_i, 0u, static_cast<u64>(k - 1), level);
        cut_key = c.key;
        ties = c.mass;
        ties_kept = min(ties, static_cast<u64>(k) - c.above);
    }
    const float p = set.top_p[row];
    if (p < 1.0f) {
        u64 mine = 0;
        for (int i = lo_i + lane; i < hi_i; i += 32) {
            const float x = at(i);
            const unsigned key = key_of(x);
            if (key > cut_key || (key == cut_key && ties == ties_kept)) mine += heat.weight(x);
        }
        mine = warp_sum64(mine);
        if (lane == 0) s.warp_sum[warp] = mine;
        __syncthreads();
        if (tid < static_cast<int>(ranks)) {
            u64 sum = 0;
            for (int w = 0; w < kWarps; ++w) sum += s.warp_sum[w];
            *cluster.map_shared_rank(&s.mass[rank], tid) = sum;
        }
        cluster.sync();
        u64 z = 0;
        for (unsigned r = 0; r < ranks; ++r) z += s.mass[r];
        const u64 w_cut = heat.weight(value_of(cut_key));
        if (ties != ties_kept) z += ties_kept * w_cut;
        const u64 target = static_cast<u64>(static_cast<double>(fmaxf(p, 0.f)) * static_cast<double>(z));
        const Cut c = find_cut<true>(cluster, s, heat, at, lo_i, hi_i, cut_key, target, level);
        const u64 w = heat.weight(value_of(c.key));
        const u64 there = c.key == cut_key && ties ? ties_kept : c.mass / w;    // tokens of that key which top-k left
        const u64 all = c.key == cut_key && ties ? ties : there;
        cut_key = c.key;
        ties = all;
        ties_kept = min(there, (target - c.above) / w + 1);
    }
    const float least = fminf(set.min_p[row], 1.0f);
    if (least > 0.f) {
        // the smallest key whose weight is min-p of the largest
        const double bound = static_cast<double>(least) * static_cast<double>(1ull << kFraction);
        if (warp == 0) {
            const unsigned lowest = first_key(key_of(-INFINITY), best, lane, [&](unsigned q) { return heat.scaled(value_of(q)) >= bound; });
            if (lane == 0) s.lo = lowest;
        }
        __syncthreads();
        if (s.lo > cut_key) {
            cut_key = s.lo;
            ties = ties_kept = 0;
        }
    }
    if (ties_kept < ties) {
        // the index of the last of the equal logits that are kept
        unsigned mine = 0;
        for (int i = lo_i + lane; i < hi_i; i += 32) mine += key_of(at(i)) == cut_key ? 1u : 0u;
        mine = __reduce_add_sync(0xffffffffu, mine);
        if (lane == 0) s.key[warp] = mine;
        __syncthreads();
        if (tid < static_cast<int>(ranks)) {
            unsigned sum = 0;
            for (int w = 0; w < kWarps; ++w) sum += s.key[w];
            *cluster.map_shared_rank(&s.ties[rank], tid) = sum;
        }
        cluster.sync();
        u64 before = 0;
        for (unsigned r = 0; r < rank; ++r) before += s.ties[r];
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
    auto kept_weight = [&](int i) -> u64 {
        const float x = at(i);
        const unsigned key = key_of(x);
        return key > cut_key || (key == cut_key && i <= tie_cut) ? heat.weight(x) : 0ull;
    };

    // ---- masses of the segments
    u64 mine = 0;
    for (int i = lo_i + lane; i < hi_i; i += 32) mine += kept_weight(i);
    mine = warp_sum64(mine);
    __syncthreads();
    if (lane == 0) s.warp_sum[warp] = mine;
    __syncthreads();
    if (tid < static_cast<int>(ranks)) {
        u64 sum = 0;
        for (int w = 0; w < kWarps; ++w) sum += s.warp_sum[w];
        *cluster.map_shared_rank(&s.total[rank], tid) = sum;
    }
    cluster.sync();
    u64 z = 0, base_mass = 0;
    for (unsigned r = 0; r < ranks; ++r) {
        if (r == rank) base_mass = z;
        z += s.total[r];
    }
    // ---- the draws: a draw whose number falls on this CTA is taken by the warp on whose segment it falls
    u64 from = base_mass;
    for (int w = 0; w < warp; ++w) from += s.warp_sum[w];
    for (int j = 0; j < draws; ++j) {
        const float u = uniform[draw0 + j];
        u64 target = u > 0.f ? static_cast<u64>(static_cast<double>(u) * static_cast<double>(z)) : 0ull;
        target = min(target, z - 1);
        if (target < from || target >= from + mine) continue;
        u64 sum = from;
        for (int base = lo_i; base < hi_i; base += 32) {
            const u64 w = base + lane < hi_i ? kept_weight(base + lane) : 0ull;
            const u64 incl = warp_scan64(w, lane) + sum;
            const unsigned over = __ballot_sync(0xffffffffu, incl > target);
            if (over) {
                const int l = __ffs(over) - 1;
                if (lane == l) {
                    out[draw0 + j] = base + lane;
                    if (prob) prob[draw0 + j] = static_cast<float>(heat.scaled(at(base + lane)) / static_cast<double>(z));
                }
                break;
            }
            sum = __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    cluster.sync();                          // no CTA leaves while another may still read its histograms
}

template <typename T>
int launch_draw(const void* logits, long long stride, int rows, int V, const Settings& set, const float* uniform, int draws,
                int* out, float* prob, cudaStream_t stream) {
    int ranks = 1;
    while (ranks < 8 && V > ranks * 4096) ranks *= 2;
    const int most = 200 * 1024;             // bytes of a slice beside the static shared memory
    const auto segment = [&](int n) { return ((V + n * kWarps - 1) / (n * kWarps) + 7) / 8 * 8; };
    while (ranks < kMaxCluster && static_cast<long long>(segment(ranks)) * kWarps * sizeof(T) > most) ranks *= 2;
    const int seg = segment(ranks);
    const long long bytes = static_cast<long long>(seg) * kWarps * sizeof(T);
    if (bytes > most || V >= 1 << 20 || static_cast<long long>(rows) * ranks > 0x7fffffffll) return SOMI_ERR_UNSUPPORTED;
    allow_smem<draw_kernel<T>>(most);
    if (ranks > 8 && cudaFuncSetAttribute(draw_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
        return SOMI_ERR_UNSUPPORTED;
    return launch_pdl_cluster(draw_kernel<T>, dim3(static_cast<unsigned>(rows) * ranks), dim3(kThreads), static_cast<size_t>(bytes),
                              static_cast<unsigned>(ranks), stream, static_cast<const T*>(logits), stride, V, seg, set, uniform,
                              draws, out, prob);
}

}  // namespace draw
}  // namespace somi

using namespace somi;

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
