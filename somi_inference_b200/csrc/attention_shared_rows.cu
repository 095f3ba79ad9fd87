// Attention of a batch whose requests share their first positions in groups, for calls of up to 16 query rows a
// key/value head (bfloat16, head sizes 64 and 128): a few single tokens.  They are bound by latency and by reading keys
// and values once, not by products.  shared_prefix.cuh says how the work is cut.  (Beside the tcgen05 kernel, for the
// entries of few rows of larger calls, it was no faster: 64 requests behind 8,192 positions took 50 us in two kernels
// and 39 in one, since a group's prefix alone is spread over more CTAs, whose parts the merge has to read.)
//
// A CTA has four warps, each with a ring of its own in shared memory: a step is 16 keys and their values
// (cp.async of 16 bytes, rows gathered through the block table, whose entry for the next step is on its way
// meanwhile), a unit is a step of every warp.  A warp computes S = Q K^T (16 rows by 16 keys) and O += P V by
// `mma.sync` m16n8k16 from registers and ldmatrix, with a maximum, a sum and 16 rows of output of its
// own, so nothing but the ends of pieces is common to the warps.  Three CTAs an SM (192 KB in flight) keep
// HBM busy across the beginnings and ends of pieces.  Keys outside the piece are not read: cp.async fills zeros.
// Measured (the device's time in a graph of calls; an eager call takes the host 16): 2 requests behind 176 positions (14 heads of 64) 6.9 us, behind
// 8,192 (28 of 128, 17 MB) 17.5: the merge's reading of a
// part from every third CTA, the ranges and the hand-over between two kernels, not HBM.
#include "mma.cuh"
#include "shared_prefix.cuh"

namespace somi {
namespace shp {

constexpr int kFewThreads = 128, kFewWarps = kFewThreads / 32, kFewKeys = 16;
__host__ __device__ constexpr int few_stages(int hd) { return hd == 128 ? 2 : 4; }
__host__ __device__ constexpr int few_smem(int hd) { return kFewWarps * few_stages(hd) * 2 * kFewKeys * hd * 2; }

template <int HD>
__global__ void __launch_bounds__(kFewThreads, 3)
shared_rows_kernel(const Batch b, const __nv_bfloat16* __restrict__ q, long long q_stride, const __nv_bfloat16* __restrict__ keys,
                   const __nv_bfloat16* __restrict__ values, float scale_log2e, Note* __restrict__ notes,
                   unsigned* __restrict__ header, Parts parts) {
    constexpr int CH = HD / 8, STAGES = few_stages(HD), TILE = kFewKeys * HD * 2;     // chunks of a row; bytes of a step's keys
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ RangeScratch scratch;
    __shared__ GroupScratch group_scratch;
    __shared__ unsigned owned[kOwned];
    __shared__ float2 state[kFewWarps][kFewRows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    unsigned char* ring = smem + warp * STAGES * 2 * TILE;

    pdl_launch_dependents();
    Raw raw;
    const Groups groups = hold_groups<kFewThreads>(b, group_scratch, raw);              // [descriptor]
    const Range range = find_range<kFewThreads>(b, groups, raw, scratch, owned);
    pdl_wait();

    Walk walk(range);
    Piece p;
    while (walk.next(b, groups, p)) {
        const int rows = p.tokens * b.per;
        const int r0 = lane >> 2;                                     // this thread's rows are r0 and r0 + 8
        // queries straight into the registers of the products' A operands
        uint32_t qf[HD / 16][4];
        {
            const int t0 = min(r0, rows - 1) / b.per, t1 = min(r0 + 8, rows - 1) / b.per;
            const __nv_bfloat16* a0 = q + (p.token0 + t0) * q_stride + static_cast<size_t>(p.kvh * b.per + min(r0, rows - 1) - t0 * b.per) * HD;
            const __nv_bfloat16* a1 = q + (p.token0 + t1) * q_stride + static_cast<size_t>(p.kvh * b.per + min(r0 + 8, rows - 1) - t1 * b.per) * HD;
            const int c = (lane & 3) * 2;
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
                qf[k][0] = *reinterpret_cast<const uint32_t*>(a0 + 16 * k + c);
                qf[k][1] = *reinterpret_cast<const uint32_t*>(a1 + 16 * k + c);
                qf[k][2] = *reinterpret_cast<const uint32_t*>(a0 + 16 * k + 8 + c);
                qf[k][3] = *reinterpret_cast<const uint32_t*>(a1 + 16 * k + 8 + c);
            }
        }
        const int t_off = p.token0 - p.x.first;
        int last[2];                                                  // the last key that a row sees
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = r0 + 8 * h;
            last[h] = r < rows ? min(p.x.key_hi - 1, p.x.pos0 + t_off + r / b.per) : -1;
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[HD / 8][4];
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
        const int* table = b.block_table + static_cast<size_t>(p.x.table) * b.bt_stride;
        const int first = p.x.base(b) + p.unit0 * p.x.unit + warp * kFewKeys, steps = p.unit1 - p.unit0;
        // the page of key `lane & 15` of step s, or -1
        auto page_of = [&](int s) {
            const int pos = first + s * p.x.unit + (lane & 15);
            return s < steps && pos >= p.x.key_lo && pos < p.x.key_hi ? table[pos / b.page_size] : -1;
        };
        int page = page_of(0);
        auto issue = [&](int s) {
            if (s < steps) {
                const int pos = first + s * p.x.unit + (lane & 15);
                const bool there = static_cast<unsigned>(page) < static_cast<unsigned>(b.num_pages);
                const int row = there ? (page * b.nkv + p.kvh) * b.page_size + pos % b.page_size : -1;
                page = page_of(s + 1);
                unsigned char* to = ring + (s % STAGES) * 2 * TILE;
#pragma unroll
                for (int i = 0; i < kFewKeys * CH / 32; ++i) {
                    const int key = (i * 32 + lane) / CH, chunk = lane % CH;
                    const int from = __shfl_sync(0xffffffffu, row, key);
                    const size_t at = static_cast<size_t>(max(from, 0)) * HD + chunk * 8;
                    const uint32_t off = swizzled_offset<HD>(key, chunk);
                    cp_async_16(smem_u32(to) + off, keys + at, from >= 0 ? 16 : 0);
                    cp_async_16(smem_u32(to) + TILE + off, values + at, from >= 0 ? 16 : 0);
                }
            }
            cp_async_commit();
        };
#pragma unroll
        for (int s = 0; s < STAGES; ++s) issue(s);
        for (int s = 0; s < steps; ++s) {
            cp_async_wait<STAGES - 1>();
            __syncwarp();
            const uint32_t ks = smem_u32(ring + (s % STAGES) * 2 * TILE), vs = ks + TILE;
            float acc[2][4] = {};
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
                uint32_t f[4];
                ldmatrix_x4(f, ks + swizzled_offset<HD>((lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
                mma_bf16_16816(acc[0], qf[k], f[0], f[1]);
                mma_bf16_16816(acc[1], qf[k], f[2], f[3]);
            }
            const int k0 = first + s * p.x.unit + (lane & 3) * 2;
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = k0 + 8 * n + (e & 1), h = e >> 1;
                    acc[n][e] = key >= p.x.key_lo && key <= last[h] ? acc[n][e] * scale_log2e : -INFINITY;
                    top[h] = fmaxf(top[h], acc[n][e]);
                }
            float keep[2];
            bool grew = false;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
                const float now = fmaxf(m[h], top[h]);
                keep[h] = now == m[h] ? 1.f : fast_exp2(m[h] - now);
                grew = grew || (now != m[h] && m[h] != -INFINITY);
                m[h] = now;
                top[h] = now == -INFINITY ? 0.f : now;                // the reference
                l[h] *= keep[h];
            }
            if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                for (int n = 0; n < HD / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][e] *= keep[e >> 1];
            }
            uint32_t pf[4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float a = fast_exp2(acc[n][2 * h] - top[h]), c = fast_exp2(acc[n][2 * h + 1] - top[h]);
                    l[h] += a + c;                                    // (of this thread's columns)
                    pf[2 * n + h] = pack_bf16(a, c);                  // (a rounding of 2^-8 of sum p |v| at most)
                }
#pragma unroll
            for (int n = 0; n < HD / 16; ++n) {
                uint32_t f[4];
                ldmatrix_x4_trans(f, vs + swizzled_offset<HD>((lane & 7) + (((lane >> 3) & 1) << 3), 2 * n + (lane >> 4)));
                mma_bf16_16816(o[2 * n], pf, f[0], f[1]);
                mma_bf16_16816(o[2 * n + 1], pf, f[2], f[3]);
            }
            __syncwarp();                                             // the stage has been read
            issue(s + STAGES);
        }
        cp_async_wait<0>();
        // ---- the warps' results joined, in the rings' place: each warp's rows, scaled to the common maximum
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if ((lane & 3) == 0) state[warp][r0 + 8 * h] = make_float2(m[h], l[h]);
        }
        __syncthreads();
        float* mine = reinterpret_cast<float*>(smem) + warp * kFewRows * HD;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float all = -INFINITY;
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) all = fmaxf(all, state[w][r0 + 8 * h].x);
            const float f = m[h] == -INFINITY ? 0.f : fast_exp2(m[h] - all);
#pragma unroll
            for (int n = 0; n < HD / 8; ++n)
                *reinterpret_cast<float2*>(mine + (r0 + 8 * h) * HD + 8 * n + (lane & 3) * 2) = make_float2(o[n][2 * h] * f, o[n][2 * h + 1] * f);
        }
        __syncthreads();
        for (int i = tid; i < rows * (HD / 4); i += kFewThreads) {
            const int row = i / (HD / 4), c = (i % (HD / 4)) * 4, t = row / b.per;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) {
                const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem) + (w * kFewRows + row) * HD + c);
                sum.x += v.x;
                sum.y += v.y;
                sum.z += v.z;
                sum.w += v.w;
            }
            const size_t at = part_row(b, p.x.pos0 == 0x3fffffff, p.first, blockIdx.x, p.token0 + t, p.kvh * b.per + row - t * b.per, row);
            *reinterpret_cast<float4*>(parts.o + at * HD + c) = sum;
            if (c == 0) {
                float all = -INFINITY, total = 0.f;
#pragma unroll
                for (int w = 0; w < kFewWarps; ++w) all = fmaxf(all, state[w][row].x);
#pragma unroll
                for (int w = 0; w < kFewWarps; ++w)
                    if (state[w][row].x != -INFINITY) total += state[w][row].y * fast_exp2(state[w][row].x - all);
                parts.ml[at] = make_float2(all, total);
            }
        }
        __syncthreads();                                              // the rings may be filled again
    }
    write_notes<kFewThreads>(b, groups, owned, range.total, notes, header, tid);
}

template <int HD>
static int launch_rows(const Batch& b, const void* q, long long q_stride, const void* keys, const void* values, float scale,
                       Note* notes, unsigned* header, Parts parts, int ctas, cudaStream_t stream) {
    allow_smem<shared_rows_kernel<HD>>(few_smem(HD));
    return launch_pdl(shared_rows_kernel<HD>, dim3(ctas), dim3(kFewThreads), few_smem(HD), stream, b,
                      static_cast<const __nv_bfloat16*>(q), q_stride, static_cast<const __nv_bfloat16*>(keys),
                      static_cast<const __nv_bfloat16*>(values), scale * 1.4426950408889634f, notes, header, parts);
}

int shared_attention_rows(Batch b, const void* q, long long q_stride, const void* keys, const void* values, int hd, float scale,
                          Note* notes, unsigned* header, Parts parts, int ctas, cudaStream_t stream) {
    b.item_tokens = b.wide_tokens = kFewRows / b.per;
    b.align = kFewKeys;
    b.unit_narrow = b.unit_wide = kFewWarps * kFewKeys;
    return hd == 64 ? launch_rows<64>(b, q, q_stride, keys, values, scale, notes, header, parts, ctas, stream)
                    : launch_rows<128>(b, q, q_stride, keys, values, scale, notes, header, parts, ctas, stream);
}

}  // namespace shp
}  // namespace somi
