// Attention of a batch whose requests share their first positions in groups, for any type and head size
// (shared_prefix.cuh says how the work is cut), and the kernel that joins the parts.
//
// A CTA holds up to 64 query rows (the query heads of a key/value head, of as many tokens as fit) in
// shared memory as float32 and walks through its pieces in tiles of 64 keys: scores and outputs by
// float32 FMAs, four rows by four columns a thread, the softmax online in float32, base 2.  It is the
// path of float32 and of head sizes and pages that the tensor-core kernel does not take.
//
// Measured (float32): 8 requests behind 1,504 positions (14 heads of 64) 19.1 us, a chain of phases (load, scores, softmax, outputs) of
// one or two tiles a CTA and the merge; portions of 40 of 24 requests behind 4,096 (28 of 128) 1,192 us, 50 TFLOP/s of the 74 that
// the FMA pipe reaches.
#include "mma.cuh"
#include "shared_prefix.cuh"
#include "vec4.cuh"

namespace somi {
namespace shp {

constexpr int kRows = 64, kKeys = 64, kThreads = 256;

// HD: the head size rounded up to 64, 128 or 256; d: the head size (a multiple of 16)
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, HD <= 128 ? 2 : 1)
shared_attention_kernel(const Batch b, const T* __restrict__ q, long long q_stride, const T* __restrict__ keys,
                        const T* __restrict__ values, int d, float scale_log2e, Note* __restrict__ notes,
                        unsigned* __restrict__ header, Parts parts) {
    constexpr int LD = HD + 4;                       // floats of a row: 16-byte reads of 8 rows meet no bank twice
    constexpr int LP = kKeys + 4;
    constexpr int COLS = HD / 16;                    // output columns of a thread
    extern __shared__ __align__(16) float smem[];
    float* Qs = smem;                                // [kRows][LD]
    float* KV = Qs + kRows * LD;                     // [kKeys][LD], keys, then values
    float* Ps = KV + kKeys * LD;                     // [kRows][LP]
    __shared__ RangeScratch scratch;

    pdl_launch_dependents();
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    __shared__ GroupScratch group_scratch;
    Raw raw;
    const Groups groups = hold_groups<kThreads>(b, group_scratch, raw);      // [descriptor]
    __shared__ unsigned owned[kOwned];
    const Range range = find_range<kThreads>(b, groups, raw, scratch, owned);
    pdl_wait();

    Walk walk(range);
    Piece p;
    while (walk.next(b, groups, p)) {
        const int rows = p.tokens * b.per;
        __syncthreads();
#pragma unroll
        for (int n = 0; n < HD / 16; ++n) {
            const int i = tid + n * kThreads, row = i / (HD / 4), c = (i % (HD / 4)) * 4, t = row / b.per;
            F4 v{{0.f, 0.f, 0.f, 0.f}};
            if (row < rows && c < d)
                v = load4(q + (p.token0 + t) * q_stride + static_cast<size_t>(p.kvh * b.per + row - t * b.per) * d + c);
            store4(Qs + row * LD + c, v);
        }
        float m[4], l[4], o[4][COLS];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.f;
#pragma unroll
            for (int c = 0; c < COLS; ++c) o[i][c] = 0.f;
        }
        int last[4];                                 // the last key that a row sees
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = ty * 4 + i;
            const int t = row / b.per + (p.token0 - p.x.first);
            last[i] = row < rows ? min(p.x.key_hi - 1, p.x.pos0 + t) : -1;
        }
        const int kb0 = p.x.base(b);
        const int* table = b.block_table + static_cast<size_t>(p.x.table) * b.bt_stride;
        // A tile of keys or values on its way to shared memory: loaded into registers while the products of the tile in front
        // are computed.  What lies outside the piece's keys, or on no page, becomes zeros.
        F4 tile[HD / 16];
        auto fetch = [&](const T* __restrict__ from, int k0) {
            const T* at[HD / 16];
#pragma unroll
            for (int n = 0; n < HD / 16; ++n) {
                const int i = tid + n * kThreads, key = i / (HD / 4), c = (i % (HD / 4)) * 4, pos = k0 + key;
                at[n] = nullptr;
                if (c < d && pos >= p.x.key_lo && pos < p.x.key_hi) {
                    const int page = table[pos / b.page_size];
                    if (static_cast<unsigned>(page) < static_cast<unsigned>(b.num_pages))
                        at[n] = from + ((static_cast<size_t>(page) * b.nkv + p.kvh) * b.page_size + pos % b.page_size) * d + c;
                }
            }
#pragma unroll
            for (int n = 0; n < HD / 16; ++n) {
                tile[n] = F4{{0.f, 0.f, 0.f, 0.f}};
                if (at[n]) tile[n] = load4(at[n]);
            }
        };
        auto put = [&]() {
#pragma unroll
            for (int n = 0; n < HD / 16; ++n) {
                const int i = tid + n * kThreads;
                store4(KV + (i / (HD / 4)) * LD + (i % (HD / 4)) * 4, tile[n]);
            }
        };
        fetch(keys, kb0 + p.unit0 * p.x.unit);
        for (int u = p.unit0; u < p.unit1; ++u) {
            const int k0 = kb0 + u * p.x.unit;
            __syncthreads();
            put();
            __syncthreads();
            fetch(values, k0);
            float s[4][4] = {};
            for (int c = 0; c < HD; c += 4) {
                F4 a[4], k[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = load4(Qs + (ty * 4 + i) * LD + c);
#pragma unroll
                for (int j = 0; j < 4; ++j) k[j] = load4(KV + (tx + 16 * j) * LD + c);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[i][j] = fmaf(a[i].v[e], k[j].v[e], s[i][j]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int pos = k0 + tx + 16 * j;
                    s[i][j] = pos >= p.x.key_lo && pos <= last[i] ? s[i][j] * scale_log2e : -INFINITY;
                    top = fmaxf(top, s[i][j]);
                }
#pragma unroll
                for (int x = 8; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                const float now = fmaxf(m[i], top);
                const float ref = now == -INFINITY ? 0.f : now;
                const float keep = exp2f(m[i] - ref);
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float w = exp2f(s[i][j] - ref);
                    sum += w;
                    Ps[(ty * 4 + i) * LP + tx + 16 * j] = w;
                }
#pragma unroll
                for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                l[i] = l[i] * keep + sum;
                m[i] = now;
#pragma unroll
                for (int c = 0; c < COLS; ++c) o[i][c] *= keep;
            }
            __syncthreads();                         // all threads have read the keys
            put();
            __syncthreads();
            if (u + 1 < p.unit1) fetch(keys, k0 + p.x.unit);
            // (a value that a row does not see stays out of its sum even if it is infinite)
            const bool all_seen = k0 + kKeys - 1 <= p.x.pos0;
            for (int j = 0; j < kKeys; j += 4) {
                F4 w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = load4(Ps + (ty * 4 + i) * LP + j);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int c = 0; c < COLS; ++c) {
                        const float v = KV[(j + e) * LD + tx + 16 * c];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (all_seen || k0 + j + e <= last[i]) o[i][c] = fmaf(w[i].v[e], v, o[i][c]);
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = ty * 4 + i;
            if (row >= rows) continue;
            const size_t at = part_row(b, p.x.pos0 == 0x3fffffff, p.first, blockIdx.x, p.token0 + row / b.per,
                                       p.kvh * b.per + row % b.per, row);
#pragma unroll
            for (int c = 0; c < COLS; ++c)
                if (tx + 16 * c < d) parts.o[at * d + tx + 16 * c] = o[i][c];
            if (tx == 0) parts.ml[at] = make_float2(m[i], l[i]);
        }
    }
    write_notes<kThreads>(b, groups, owned, range.total, notes, header, tid);
}

// What a row that is not finite is computed again from.  `q` null: never.
template <typename T>
struct Source {
    const T *q, *keys, *values;
    long long q_stride;
    float scale_log2e;
};

// A row by itself, over the keys that it sees and nothing else; by one warp, four columns a lane (head sizes to 128).  The
// tensor-core kernels multiply a value that a row does not see by a probability of 0, and where that value is infinite or not a
// number the row is lost.  Only a later token of the row's own portion can do that, so nothing is computed where no such token
// has such a value.  (Few registers rather than many loads in flight: behind 20,000 positions a row takes 20 ms, but the merge keeps
// its eight blocks an SM, without which 24 portions took 168 us for 163.)
template <typename T>
__device__ __noinline__ void row_alone(const Batch& b, const Source<T>& from, int d, int t, int h, T* out) {
    const int lane = threadIdx.x & 31, c = lane * 4, kvh = h / b.per;
    int r = 0;
    for (int hi = b.R - 1; r < hi;) {                // the last request that begins at or in front of t
        const int mid = (r + hi + 1) >> 1;
        if (b.cu_q[mid] <= t) r = mid;
        else hi = mid - 1;
    }
    const int span = b.bt_stride * b.page_size, ctx = clamped(b.ctx_len[r], 0, span);
    const int pos = min(ctx + t - b.cu_q[r], span - 1), end = min(ctx + b.cu_q[r + 1] - b.cu_q[r], span);
    const int* table = b.block_table + static_cast<size_t>(r) * b.bt_stride;
    auto row_of = [&](const T* store, int key) {
        const int page = table[key / b.page_size];
        F4 v{{0.f, 0.f, 0.f, 0.f}};
        if (c < d && static_cast<unsigned>(page) < static_cast<unsigned>(b.num_pages))
            v = load4(store + ((static_cast<size_t>(page) * b.nkv + kvh) * b.page_size + key % b.page_size) * d + c);
        return v;
    };
    bool lost = false;
    for (int key = pos + 1; key < end; ++key) {
        const F4 v = row_of(from.values, key);
#pragma unroll
        for (int e = 0; e < 4; ++e) lost = lost || !isfinite(v.v[e]);
    }
    if (!__any_sync(0xffffffffu, lost)) return;
    F4 q{{0.f, 0.f, 0.f, 0.f}}, o = q;
    if (c < d) q = load4(from.q + t * from.q_stride + static_cast<size_t>(h) * d + c);
    float m = -INFINITY, l = 0.f;
    constexpr int AT_ONCE = 2;
    for (int k0 = 0; k0 <= pos; k0 += AT_ONCE) {
        float s[AT_ONCE], top = m;
        F4 v[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const F4 k = row_of(from.keys, min(k0 + i, pos));
            v[i] = row_of(from.values, min(k0 + i, pos));
            s[i] = fmaf(q.v[3], k.v[3], fmaf(q.v[2], k.v[2], fmaf(q.v[1], k.v[1], q.v[0] * k.v[0])));
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            s[i] = k0 + i <= pos ? warp_sum(s[i]) * from.scale_log2e : -INFINITY;
            top = fmaxf(top, s[i]);
        }
        const float ref = top == -INFINITY ? 0.f : top, keep = exp2f(m - ref);
        m = top;
        l *= keep;
#pragma unroll
        for (int e = 0; e < 4; ++e) o.v[e] *= keep;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            if (k0 + i > pos) continue;
            const float w = exp2f(s[i] - ref);
            l += w;
#pragma unroll
            for (int e = 0; e < 4; ++e) o.v[e] = fmaf(w, v[i].v[e], o.v[e]);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.v[e] *= inv;
    if (c < d) store4(out + (static_cast<size_t>(t) * b.nq + h) * d + c, o);
}

constexpr int kFewRowsOut = 4 * 148;     // four blocks an SM

// SPLIT warps per (token, head), a block of WARPS.  A lane finds out where a part lies and loads its maximum and sum, for
// up to 32 parts at once; then all lanes add the parts' outputs up, several loads in flight.  The parts go round the row's
// warps, whose sums are joined in shared memory.
template <typename T, int WARPS, int SPLIT>
__global__ void __launch_bounds__(WARPS * 32)
shared_merge_kernel(const __grid_constant__ Batch b, int d, const Note* __restrict__ notes, const unsigned* __restrict__ header, Parts parts,
                    int ctas, const __grid_constant__ Source<T> from, T* __restrict__ out) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int warp = (threadIdx.x >> 5) % SPLIT;
    const long long row = static_cast<long long>(blockIdx.x) * (WARPS / SPLIT) + (threadIdx.x >> 5) / SPLIT;
    static_assert(SPLIT == 1 || SPLIT == WARPS, "the returns below are the whole block's where it joins its warps");
    if (row >= static_cast<long long>(b.T) * b.nq) return;
    const int t = static_cast<int>(row / b.nq), h = static_cast<int>(row % b.nq), kvh = h / b.per;
    const unsigned total = header[0];
    const Note prefix = notes[t], own = notes[b.T + t];              // (the first may be unwritten)
    if (b.cu_q && (t < b.cu_q[0] || t >= b.cu_q[b.R])) return;       // a row of no request stays as it was
    if (total == 0) return;
    const Shares shares(total, ctas);
    // the CTAs that had a part of an item, neighbours all
    struct Item { unsigned begin, first_cta, ctas; int place; };
    auto item_of = [&](const Note& n, bool written) {
        Item x;
        x.place = n.place & ~kHasPrefix;
        x.begin = n.begin + static_cast<unsigned>(kvh) * n.cost;
        const unsigned end = x.begin + n.cost;
        // (the second half: what no note of a request's token looks like)
        const bool there = written && n.units > 0 && n.cost > n.units && end <= total && end >= x.begin && x.place >= 0 &&
                           (x.place + 1) * b.per <= b.block_rows;
        x.first_cta = there ? shares.cta_of(x.begin) : 0u;
        x.ctas = there ? shares.cta_of(end - 1) - x.first_cta + 1 : 0u;
        return x;
    };
    const Item front = item_of(prefix, own.place & kHasPrefix), back = item_of(own, true);
    const unsigned all = front.ctas + back.ctas;
    constexpr int COLS = 2;                          // of four columns a lane: head sizes to 256
    float m = -INFINITY, l = 0.f;
    F4 o[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) o[c] = F4{{0.f, 0.f, 0.f, 0.f}};
    for (unsigned p0 = 0; p0 < all; p0 += 32 * SPLIT) {
        const unsigned p = p0 + lane * SPLIT + warp;
        size_t at = 0;
        float2 ml = make_float2(-INFINITY, 0.f);
        if (p < all) {
            const bool first = p < front.ctas;
            const unsigned begin = first ? front.begin : back.begin, cost = first ? prefix.cost : own.cost;
            const unsigned over = cost - static_cast<unsigned>(first ? prefix.units : own.units);
            const unsigned cta = first ? front.first_cta + p : back.first_cta + p - front.ctas;
            const unsigned c0 = shares.begin(cta), c1 = shares.begin(cta + 1);
            const unsigned o0 = c0 > begin ? c0 - begin : 0, o1 = min(c1 - begin, cost);
            if (o1 > over && o1 > o0) {  // (else it had only the item's fixed cost)
                at = part_row(b, first, o0 == 0, cta, t, h, (first ? front.place : back.place) * b.per + h % b.per);
                ml = parts.ml[at];
            }
        }
        const bool some = !(ml.x == -INFINITY && ml.y == 0.f);      // (a part whose keys are all hidden has no output)
        const float now = fmaxf(m, warp_max(ml.x)), ref = now == -INFINITY ? 0.f : now;
        const float keep = exp2f(m - ref), weight = some ? exp2f(ml.x - ref) : 0.f;
        l = l * keep + warp_sum(some ? ml.y * weight : 0.f);
        m = now;
#pragma unroll
        for (int c = 0; c < COLS; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[c].v[e] *= keep;
        const unsigned live = __ballot_sync(0xffffffffu, some);
        for (unsigned left = live; left != 0;) {
            // up to four parts at a time
            F4 v[4][COLS];
            float w[4];
            unsigned rest = left;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int from = rest ? __ffs(rest) - 1 : 0;
                const size_t where = __shfl_sync(0xffffffffu, static_cast<unsigned long long>(at), from);
                w[k] = __shfl_sync(0xffffffffu, weight, from);
#pragma unroll
                for (int c = 0; c < COLS; ++c)
                    if (rest && (c * 32 + lane) * 4 < d) v[k][c] = load4(parts.o + where * d + (c * 32 + lane) * 4);
                    else v[k][c] = F4{{0.f, 0.f, 0.f, 0.f}};
                if (!rest) w[k] = 0.f;
                rest &= rest - 1;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int c = 0; c < COLS; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[c].v[e] = fmaf(v[k][c].v[e], w[k], o[c].v[e]);
            left = rest;
        }
    }
    if constexpr (SPLIT > 1) {
        __shared__ float2 state[SPLIT];
        __shared__ __align__(16) float rows[SPLIT][256];
        if (lane == 0) state[warp] = make_float2(m, l);
#pragma unroll
        for (int c = 0; c < COLS; ++c)
            if ((c * 32 + lane) * 4 < d) store4(&rows[warp][(c * 32 + lane) * 4], o[c]);
        __syncthreads();
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < SPLIT; ++w) top = fmaxf(top, state[w].x);
        const float ref = top == -INFINITY ? 0.f : top;
        float f[SPLIT];
#pragma unroll
        for (int w = 0; w < SPLIT; ++w) {
            f[w] = exp2f(state[w].x - ref);
            sum = fmaf(state[w].y, f[w], sum);
        }
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        bool lost = false;
        for (int col = threadIdx.x; col < d; col += WARPS * 32) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < SPLIT; ++w) v = fmaf(rows[w][col], f[w], v);
            out[row * d + col] = from_float<T>(v * inv);
            lost = lost || !isfinite(v * inv);
        }
        if (from.q && __syncthreads_or(lost) && threadIdx.x < 32) row_alone(b, from, d, t, h, out);
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    bool lost = false;
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
        const int col = (c * 32 + lane) * 4;
        if (col < d) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                o[c].v[e] *= inv;
                lost = lost || !isfinite(o[c].v[e]);
            }
            store4(out + row * d + col, o[c]);
        }
    }
    if (from.q && __any_sync(0xffffffffu, lost)) row_alone(b, from, d, t, h, out);
}

template <typename T, int HD>
int launch_shared(const Batch& b, const void* q, long long q_stride, const void* keys, const void* values, int d, float scale,
                  Note* notes, unsigned* header, Parts parts, int ctas, cudaStream_t stream) {
    constexpr int smem = (kRows * (HD + 4) + kKeys * (HD + 4) + kRows * (kKeys + 4)) * 4;
    allow_smem<shared_attention_kernel<T, HD>>(smem);
    return launch_pdl(shared_attention_kernel<T, HD>, dim3(ctas), dim3(kThreads), smem, stream, b,
                      static_cast<const T*>(q), q_stride, static_cast<const T*>(keys), static_cast<const T*>(values), d,
                      scale * 1.4426950408889634f, notes, header, parts);
}

}  // namespace shp
}  // namespace somi

using namespace somi;
using namespace somi::shp;

// The kernels: 0 the one for any size, 1 the one on tensor cores, 2 that for few rows.  CTAs, and the rows of one CTA's continuation.
SOMI_API int somi_shared_attention_ctas(int hd, int kernel) {
    int device = 0, sms = 0;
    cudaGetDevice(&device);
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms <= 0) return 0;
    return sms * (kernel == 2 ? 3 : kernel == 1 ? 1 : hd <= 64 ? 4 : hd <= 128 ? 2 : 1);
}
SOMI_API int somi_shared_attention_block_rows(int kernel) {
    return kernel == 2 ? kFewRows : kernel == 1 ? somi_shared_attention_tc_block_rows() : kRows;
}

// Bytes of workspace: notes, the header, maxima and sums, outputs.
static long long workspace_bytes(long long T, long long rows, int hd) {
    return 2 * T * static_cast<long long>(sizeof(Note)) + 32 + rows * 8 + rows * hd * 4;
}

// qkv [T, >= nq hd] (rows `q_stride` elements apart), keys and values [num_pages, nkv, page_size, hd], block_table
// [R, bt_stride], cu_q [R + 1] or null (then T = R, one token per request), ctx_len [R], group_off [G + 1], prefix_len [G];
// `out` [T, nq hd].  `kernel`: see above (1 and 2 where somi_shared_attention_tc_takes says so, 2 for at most 16 rows a
// key/value head).  Refuses what it cannot take; the lengths are read on the device.
SOMI_API int somi_shared_attention(const void* qkv, int dtype, long long q_stride, const void* keys, const void* values,
                                   const int* block_table, int bt_stride, const int* cu_q, const int* ctx_len,
                                   const int* prefix_len, const int* group_off, int T, int R, int G, int nq, int nkv, int hd,
                                   int page_size, int num_pages, float scale, int kernel, void* workspace, long long bytes,
                                   int ctas, void* out, cudaStream_t stream) {
    if (T <= 0 || R <= 0) return 0;
    if (nkv <= 0 || nq <= 0 || nq % nkv || (!kernel && nq / nkv > kRows) || hd % 16 || hd < 16 || hd > 256 || G < 0 || bt_stride <= 0 ||
        page_size <= 0 || num_pages <= 0 || kernel < 0 || kernel > 2 || ctas <= 0 || static_cast<long long>(R) + G > kMaxEntries ||
        static_cast<long long>(R) + G > static_cast<long long>(ctas) * kOwned || (!cu_q && T != R))
        return SOMI_ERR_UNSUPPORTED;
    const int per = nq / nkv;
    if (kernel && (dtype != SOMI_BF16 || !somi_shared_attention_tc_takes(nq, nkv, hd, page_size))) return SOMI_ERR_UNSUPPORTED;
    if (kernel == 1 && !(scale > 0.f)) return SOMI_ERR_UNSUPPORTED;      // (it scales a row's maximum, and hidden scores)
    if (kernel == 2 && static_cast<long long>(T) * per > kFewRows) return SOMI_ERR_UNSUPPORTED;
    const long long span = static_cast<long long>(bt_stride) * page_size;
    const int block_rows = somi_shared_attention_block_rows(kernel);
    const int item_tokens = (kernel == 1 ? block_rows / 2 : block_rows) / per;
    const long long items = (R + static_cast<long long>(G) + 2 * (T / item_tokens + 1ll)) * nkv;
    if (span > 0x3fff0000ll || items * (span / kKeys + 3) > 0x7fffffffll || static_cast<long long>(T) * nq >= 0x1fffffffcll ||
        static_cast<long long>(num_pages) * nkv * page_size > 0x7fffffffll)
        return SOMI_ERR_UNSUPPORTED;
    const long long rows = 2ll * T * nq + static_cast<long long>(ctas) * block_rows;
    if (reinterpret_cast<uintptr_t>(workspace) % 32) return SOMI_ERR_UNSUPPORTED;
    if (bytes < workspace_bytes(T, rows, hd)) return SOMI_ERR_SCRATCH_TOO_SMALL;
    const Batch b{cu_q, ctx_len, prefix_len, group_off, block_table, bt_stride, R, G, T, nq, nkv, per, page_size, num_pages,
                  item_tokens, item_tokens, kKeys, kKeys, kKeys, 1, block_rows};
    char* at = static_cast<char*>(workspace);
    Note* notes = reinterpret_cast<Note*>(at);
    unsigned* header = reinterpret_cast<unsigned*>(at + 2ll * T * sizeof(Note));
    Parts parts;
    parts.o = reinterpret_cast<float*>(header + 8);      // (on a boundary of 32 bytes, as the workspace is)
    parts.ml = reinterpret_cast<float2*>(parts.o + rows * hd);
    const auto launch = [&](auto kind) {
        using E = decltype(kind);
        const int rc =
            kernel == 2 ? shared_attention_rows(b, qkv, q_stride, keys, values, hd, scale, notes, header, parts, ctas, stream)
            : kernel == 1 ? shared_attention_tc(b, qkv, q_stride, keys, values, hd, scale, notes, header, parts, ctas, stream)
            : hd <= 64    ? launch_shared<E, 64>(b, qkv, q_stride, keys, values, hd, scale, notes, header, parts, ctas, stream)
            : hd <= 128   ? launch_shared<E, 128>(b, qkv, q_stride, keys, values, hd, scale, notes, header, parts, ctas, stream)
                          : launch_shared<E, 256>(b, qkv, q_stride, keys, values, hd, scale, notes, header, parts, ctas, stream);
        if (rc) return rc;
        // (the kernel for any size keeps out what a row does not see, and a single token has no later ones)
        const Source<E> from{kernel && cu_q ? static_cast<const E*>(qkv) : nullptr, static_cast<const E*>(keys),
                             static_cast<const E*>(values), q_stride, scale * 1.4426950408889634f};
        const long long out_rows = static_cast<long long>(T) * nq;
        // Few rows have their keys in many CTAs.  One warp a row against eight: 2 requests behind 8,192 positions 32.4 us and
        // 12.5 (14 heads of 64), 8 behind 2,048 14.5 and 13.5 (28 of 128), 32 behind 4,096 19.4 and 16.4 (448 rows), but 896 rows
        // 22.8 and 25.1.  Up to 8 steps of 64 keys there is nothing to divide (2 behind 176: 7.0 and 7.3).
        if (out_rows <= kFewRowsOut && span > 512)
            return launch_pdl(shared_merge_kernel<E, 8, 8>, dim3(static_cast<unsigned>(out_rows)), dim3(256), 0, stream, b, hd, notes,
                              header, parts, ctas, from, static_cast<E*>(out));
        return launch_pdl(shared_merge_kernel<E, 4, 1>, dim3(static_cast<unsigned>((out_rows + 3) / 4)), dim3(128), 0, stream, b, hd,
                          notes, header, parts, ctas, from, static_cast<E*>(out));
    };
    return dtype == SOMI_F32 ? launch(float{}) : dtype == SOMI_BF16 ? launch(__nv_bfloat16{}) : SOMI_ERR_UNSUPPORTED;
}
