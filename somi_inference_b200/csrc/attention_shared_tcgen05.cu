// Attention of a batch whose requests share their first positions in groups, on the 5th-generation tensor
// cores (bfloat16, head sizes 64 and 128).  shared_prefix.cuh says how the work is cut into pieces: up to 256
// query rows (the heads of a key/value head, of as many tokens as fit) over a range of key tiles of 128.
//
// A CTA has two softmax warp groups, A and B, each with scores S and outputs O of its own in tensor memory
// (128 lanes: a row each).  A piece is computed in one of two ways:
//     wide    (more rows than 128): A and B hold 128 rows each and work on the same key tile, which is
//             fetched once for both;
//     narrow  (up to 128 rows): A and B hold the same rows and take key tiles in turn; at the end of the piece their
//             outputs are joined like any two parts.  So few rows use both warp groups, too, and have twice
//             as many keys in flight.
// Both products are `tcgen05.mma`: S = Q K^T from shared memory; the probabilities are written over S as bfloat16 pairs
// and are the tensor-memory A operand of O += P V (rounding P to bfloat16 moves the output by at most 2^-8 of
// sum p |v|, the same as the other tensor-core kernels; its sum l is taken in float32 before).  While one warp group computes
// probabilities the tensor cores run the other's products.
//
// Warp roles: 0-3 softmax A, 4-7 softmax B (they also gather the queries, whose rows lie scattered over
// tokens and heads, into the swizzled shared-memory layout, and write the parts), 8 key producer, 9 MMA issuer,
// 10 value producer, 11 walks through the CTA's pieces and writes them into a ring, so that what a piece
// needs from the lengths' arrays has been read before anybody waits for it.  Key and value stages lie in one
// pool: wide pieces use it as one ring of keys and one of values, narrow ones as a ring for each warp group (a ring that
// is waited on by parity must be seen by its readers in every phase, which a reader of every second tile
// of a common ring would not do); the producers wait for the products of the last piece where the way changes.
//
// A value row outside the piece's keys may be anything, not a number among it: the softmax warps clear such rows
// of the first and last tile before they announce the probabilities.  Every wait on an mbarrier is
// bounded and failure is recorded in an error word.
//
// Measured (28 heads of 128 over 4), the device's time in a graph of calls: 64 requests behind 8,192 positions with up to 511 of their
// own 35.1 us, 8 behind 2,048 13.2, portions of 1 to 47 tokens of 24 requests behind 20,000 164 us (920 TFLOP/s); as calls one behind
// the other 35.4, 16.3 (the host's time) and 181 us (830 TFLOP/s).  Long pieces are bound by the softmax
// chain of a tile (load, maximum, 2^x, store: 2.1 us a pair of tiles), short ones by the chain from the block table to the
// written part (4.5 us, of which the products are a tenth).
#include "shared_prefix.cuh"
#include "tcgen05.cuh"

namespace somi {
namespace shp {

constexpr int kTcThreads = 384, kTile = 128;          // rows of a warp group; keys of a tile
constexpr int kTcBlockRows = 2 * kTile;
// An item of more than 128 rows gathers 256 rows of queries and writes 256 of outputs, and often comes between pieces of the other way:
// with a cost of 3 beside its units, where one of few rows has 1, 24 portions of 1 to 47 tokens behind 20,000 positions take 184 us (1: 278,
// 2: 213, 4: 166, 6: 169; lengths drawn anew), 16 of 100 behind 4,096 148 (1: 232, 2: 177, 4: 143, 6: 148), 60 of 1 to 20 behind 2,000
// 55.1 (58.7, 56.4, 61.2, 60.8), 8 of 60 behind 1,024 36.0 (38.1, 37.7, 36.9, 38.5); single tokens differ by 0.6 at most.
constexpr int kOverWide = 3;
constexpr int kPieces = 4;                            // of the ring of pieces
constexpr int kHalf = kTile * 128;                    // bytes of a [128][64] swizzled block
__host__ __device__ constexpr int k_stages(int hd) { return hd == 128 ? 2 : 4; }
__host__ __device__ constexpr int v_stages_wide(int hd) { return hd == 128 ? 3 : 8; }
__host__ __device__ constexpr int v_stages_narrow(int hd) { return hd == 128 ? 4 : 8; }   // (128: the second query tile's place)
constexpr int kMaxK = 4, kMaxV = 8;

__device__ int g_shared_error = 0;

// Eight floats at once, a whole sector of L2: a thread that writes a row by itself has no neighbours to fill it up.
__device__ __forceinline__ void store8(float* to, const float* v) {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(to), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
                 "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
}

// 16 columns of the thread's row, arrived.  (The wait is in the same statement: between a load and its wait the registers
// are the tensor memory's, and a compiler that copied or reused them there would not know.)
__device__ __forceinline__ void ld16(uint32_t taddr, float* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        "tcgen05.wait::ld.sync.aligned;\n"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]),
          "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(taddr)
        : "memory");
}

// All 128 columns, arrived.
__device__ __forceinline__ void ld128(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x128.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
        "%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,"
        "%54,%55,%56,%57,%58,%59,%60,%61,%62,%63,%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,"
        "%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,%96,%97,%98,%99,%100,%101,%102,%103,%104,"
        "%105,%106,%107,%108,%109,%110,%111,%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,"
        "%126,%127}, [%128];\n"
        "tcgen05.wait::ld.sync.aligned;\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]),
          "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]),
          "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]),
          "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]),
          "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]), "=r"(r[72]),
          "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]), "=r"(r[80]), "=r"(r[81]),
          "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]), "=r"(r[88]), "=r"(r[89]), "=r"(r[90]),
          "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]), "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]),
          "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]), "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]),
          "=r"(r[108]), "=r"(r[109]), "=r"(r[110]), "=r"(r[111]), "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]),
          "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]), "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]),
          "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
        : "r"(taddr)
        : "memory");
}

struct PieceNote {
    int tiles;                                        // key tiles; < 0: no more pieces
    int key0, key_lo, key_hi;                         // first key of the first tile; keys there are
    int pos0;                                         // position of the first token (prefix: all is seen)
    int token0, tokens, table, kvh;
    int wide, changed, prefix, first;
};

// What lies behind the tiles in shared memory.  Stage barriers: wide rings use [1][stage], narrow ones
// [0][x * (stages of a warp group) + stage].
struct Tail {
    unsigned long long k_full[2][kMaxK], k_empty[2][kMaxK], v_full[2][kMaxV], v_empty[2][kMaxV];
    unsigned long long s_full[2], p_full[2], q_full, o_done, mode_done, piece_full[kPieces], piece_empty[kPieces];
    float2 b_state[kTile];                            // B's maximum and sum of each row, and A's maximum
    float a_top[kTile];
    PieceNote ring[kPieces];
    GroupScratch groups;
    unsigned owned[kOwned];
    uint32_t tmem_base;
    int failed, softmax_failed[2];
};
__host__ __device__ constexpr int tc_smem(int hd) {
    return (2 + k_stages(hd) + v_stages_wide(hd)) * (hd / 64) * kHalf + static_cast<int>(sizeof(Tail));
}
static_assert(tc_smem(128) <= 227 * 1024 && tc_smem(64) <= 227 * 1024, "more shared memory than a CTA can have");

template <int HD>
__global__ void __launch_bounds__(kTcThreads, 1)
shared_attention_tc_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Batch b,
                           const __nv_bfloat16* __restrict__ q, long long q_stride, float scale_log2e,
                           Note* __restrict__ notes, unsigned* __restrict__ header, Parts parts) {
    constexpr int HALVES = HD / 64, TILE = HALVES * kHalf;
    constexpr int KST = k_stages(HD), VSW = v_stages_wide(HD);
    constexpr int KSN = KST / 2, VSN = v_stages_narrow(HD) / 2;       // of one warp group's ring
    constexpr uint32_t TmemCols = 512;                                // S_A | S_B | O_A | O_B, 128 columns each
    extern __shared__ __align__(1024) unsigned char base[];
    unsigned char* Qs = base;
    unsigned char* Ks = Qs + TILE;                                    // KST tiles
    unsigned char* Vs = Ks + KST * TILE;                              // VSW tiles (narrow: VSN of A, VSN of B)
    unsigned char* Q1 = Vs + VSW * TILE;
    Tail& tail = *reinterpret_cast<Tail*>(Q1 + TILE);
    auto& k_full = tail.k_full; auto& k_empty = tail.k_empty; auto& v_full = tail.v_full; auto& v_empty = tail.v_empty;
    auto& s_full = tail.s_full; auto& p_full = tail.p_full; auto& ring = tail.ring;
    auto& q_full = tail.q_full; auto& o_done = tail.o_done; auto& mode_done = tail.mode_done;
    auto& piece_full = tail.piece_full; auto& piece_empty = tail.piece_empty;
    auto& tmem_base_s = tail.tmem_base; auto& failed_s = tail.failed;
    RangeScratch& scratch = *reinterpret_cast<RangeScratch*>(Vs);     // until the first copies

    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // (a thread each: one alone would keep the others waiting)
    if (tid < 4 * (kMaxK + kMaxV)) {
        unsigned long long* const barriers = &k_full[0][0];           // k_full, k_empty, v_full, v_empty, one behind the other
        mbar_init(smem_u32(barriers + tid), 1);
    } else if (tid >= 64 && tid < 64 + kPieces) {
        mbar_init(smem_u32(&piece_full[tid - 64]), 1);
        mbar_init(smem_u32(&piece_empty[tid - 64]), 11);              // 8 softmax warps, 2 producers, the issuer
    } else if (tid == 96 || tid == 97) {
        mbar_init(smem_u32(&s_full[tid - 96]), 1);
        mbar_init(smem_u32(&p_full[tid - 96]), 4);                    // one arrival per warp of the group
    } else if (tid == 128) {
        mbar_init(smem_u32(&q_full), 8);
        mbar_init(smem_u32(&o_done), 1);
        mbar_init(smem_u32(&mode_done), 1);
        failed_s = smem_u32(base) & 1023 ? 1 : 0;                     // (the swizzled layout needs the alignment)
        tail.softmax_failed[0] = tail.softmax_failed[1] = 0;
    }
    if (tid < 160) mbar_fence_init();
    static_assert(4 * (kMaxK + kMaxV) <= 64 && offsetof(Tail, s_full) == 4 * (kMaxK + kMaxV) * sizeof(unsigned long long),
                  "the rings' barriers lie one behind the other");
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_base_s)),
                     "r"(TmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    Raw raw;
    const Groups groups = hold_groups<kTcThreads>(b, tail.groups, raw);                // [descriptor]
    const Range range = find_range<kTcThreads>(b, groups, raw, scratch, tail.owned);   // [descriptor]
    t5::fence_before();
    __syncthreads();
    t5::fence_after();
    pdl_wait();
    fence_proxy_async();                                              // (the scratch lies where copies will arrive)
    __syncthreads();
    const uint32_t tmem_s = tmem_base_s, tmem_o = tmem_base_s + 2 * kTile;
    const int per_tile = kTile / b.per;                               // tokens of a warp group

    // (the launch's registers, 12 warps of 168 a thread, shared out anew: setmaxnreg.inc waits for what it asks for)
    static_assert(8 * 216 + 4 * 72 <= 12 * 168, "setmaxnreg would wait for registers that never come");
    auto get_piece = [&](int n, bool ok) -> bool {                    // by whole warps
        return mbar_wait(smem_u32(&piece_full[n % kPieces]), (n / kPieces) & 1, ok ? 400000 : 1) && ok;
    };
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
        if (warp == 11) {
            // ---- the pieces, one after the other
            Walk walk(range);
            Piece p;
            int last_wide = -1;
            bool more = true, ok = true;
            for (int n = 0; more && ok; ++n) {
                more = walk.next(b, groups, p);
                ok = mbar_wait(smem_u32(&piece_empty[n % kPieces]), ((n / kPieces) & 1) ^ 1);
                if (!ok) failed_s = 1;
                if (lane == 0) {
                    PieceNote& to = ring[n % kPieces];
                    to.tiles = -1;
                    if (more) {
                        const int wide = p.x.tokens > b.wide_tokens ? 1 : 0, step = p.x.unit / kTile;
                        // tiles behind the last key that the last token sees are left out
                        const int t_off = p.token0 - p.x.first;
                        const int end = min(p.x.key_hi, min(p.x.pos0, p.x.key_hi) + t_off + p.tokens);
                        const int b0 = p.x.base(b);
                        const int t0 = p.unit0 * step, t1 = min(p.unit1 * step, (end - b0 + kTile - 1) / kTile);
                        to.tiles = max(t1 - t0, 0);
                        const bool counts = to.tiles > 0;             // (a piece without tiles changes nothing)
                        to.key0 = b0 + t0 * kTile;
                        to.key_lo = p.x.key_lo;
                        to.key_hi = p.x.key_hi;
                        to.pos0 = p.x.pos0 + t_off;
                        to.token0 = p.token0;
                        to.tokens = p.tokens;
                        to.table = p.x.table;
                        to.kvh = p.kvh;
                        to.wide = wide;
                        to.changed = counts && last_wide >= 0 && last_wide != wide;
                        to.prefix = p.x.pos0 == 0x3fffffff;
                        to.first = p.first;
                        if (counts) last_wide = wide;
                    }
                    mbar_arrive(smem_u32(&piece_full[n % kPieces]));
                }
                __syncwarp();
            }
            // (what the merge wants to know: while the others work on the last pieces)
            write_notes<32>(b, groups, tail.owned, range.total, notes, header, lane);
        } else if (warp == 8 || warp == 10) {
            // ---- producers of keys and of values: lane 0 keeps the barriers, a lane per page copies it
            const int which = warp == 8 ? 0 : 1;
            const CUtensorMap* map = which ? &v_map : &k_map;
            unsigned char* const pool = which ? Vs : Ks;
            const int pages_per_tile = kTile / b.page_size;
            int wide_at = 0, narrow_at[2] = {0, 0}, changes = 0;
            bool ok = true;
            for (int n = 0; ok; ++n) {
                ok = get_piece(n, ok);
                const PieceNote p = ring[n % kPieces];
                if (!ok || p.tiles < 0) break;
                if (p.changed) {
                    ok = mbar_wait(smem_u32(&mode_done), changes & 1);
                    ++changes;
                }
                const int* table = b.block_table + static_cast<size_t>(p.table) * b.bt_stride;
                for (int t = 0; t < p.tiles && ok; ++t) {
                    const int kb = p.key0 + t * kTile;
                    const int pos = kb + lane * b.page_size;
                    int page = -1;
                    if (lane < pages_per_tile && pos < p.key_hi && pos + b.page_size > p.key_lo) page = ld_step(table + pos / b.page_size);
                    const bool mine = static_cast<unsigned>(page) < static_cast<unsigned>(b.num_pages);
                    const int n_pages = __popc(__ballot_sync(0xffffffffu, mine));
                    int st, round;
                    if (p.wide) {
                        const int ring_size = which ? VSW : KST;
                        st = wide_at % ring_size;
                        round = wide_at / ring_size;
                        ++wide_at;
                    } else {
                        const int x = t & 1, ring_size = which ? VSN : KSN;
                        st = x * ring_size + narrow_at[x] % ring_size;
                        round = narrow_at[x] / ring_size;
                        ++narrow_at[x];
                    }
                    unsigned long long* full = which ? &v_full[p.wide][st] : &k_full[p.wide][st];
                    unsigned long long* empty = which ? &v_empty[p.wide][st] : &k_empty[p.wide][st];
                    int good = 1;
                    if (lane == 0) {
                        good = mbar_wait(smem_u32(empty), (round & 1) ^ 1) ? 1 : 0;
                        if (good) mbar_expect_tx(smem_u32(full), static_cast<uint32_t>(n_pages) * b.page_size * HD * 2);
                    }
                    ok = __shfl_sync(0xffffffffu, good, 0) != 0;
                    if (ok && mine) {
                        const int row = (page * b.nkv + p.kvh) * b.page_size;
                        unsigned char* dst = pool + st * TILE + lane * b.page_size * 128;
#pragma unroll
                        for (int h = 0; h < HALVES; ++h)
                            tma_load_2d(smem_u32(dst + h * kHalf), map, h * 64, row, smem_u32(full));
                    }
                }
                __syncwarp();
                if (ok && lane == 0) mbar_arrive(smem_u32(&piece_empty[n % kPieces]));
            }
            if (!ok) failed_s = 1;
        } else if (lane == 0) {
            // ---- issuer: float32 accumulators, bf16 operands; scores A and B K-major, N = 128 keys;
            // outputs A from tensor memory, B (V) MN-major, N = head size
            const uint32_t idesc_qk = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(kTile >> 3) << 17) |
                                      (static_cast<uint32_t>(kTile >> 4) << 24);
            const uint32_t idesc_pv = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (static_cast<uint32_t>(HD >> 3) << 17) |
                                      (static_cast<uint32_t>(kTile >> 4) << 24);
            const uint64_t q_desc = t5::desc_kmajor(smem_u32(Qs));
            const uint64_t k_desc = t5::desc_kmajor(smem_u32(Ks));
            const uint64_t v_desc = t5::desc_mnmajor(smem_u32(Vs), kHalf);
            bool ok = true;
            auto wait = [&](unsigned long long* bar, int parity) {
                if (ok && !mbar_wait(smem_u32(bar), parity)) ok = false;
                t5::fence_after();
            };
            auto spin = [&](unsigned long long* bar, int parity) {
                if (ok) {
                    int i = 0;
                    while (!mbar_test_now(smem_u32(bar), parity))
                        if (++i > 8000000) { ok = false; break; }
                }
                t5::fence_after();
            };
            int wide_at = 0, narrow_a = 0, narrow_b = 0;              // tiles of the pieces before
            int done_a = 0, done_b = 0;                               // rounds of the warp groups before
            for (int n = 0; ok; ++n) {
                wait(&piece_full[n % kPieces], (n / kPieces) & 1);
                if (!ok) break;
                const int nt = ring[n % kPieces].tiles, wide = ring[n % kPieces].wide;
                if (nt < 0) break;
                if (ring[n % kPieces].changed) t5::commit(smem_u32(&mode_done));
                const int nx0 = wide ? nt : (nt + 1) / 2, nx1 = wide ? (ring[n % kPieces].tokens > per_tile ? nt : 0) : nt / 2;
                mbar_arrive(smem_u32(&piece_empty[n % kPieces]));
                wait(&q_full, n & 1);
                // (one copy of each product in the code: this warp has few registers)
                for (int i = -1; i < nx0 && ok; ++i) {
#pragma unroll 1
                    for (int x = 0; x < 2; ++x) {
                        const int n_x = x ? nx1 : nx0;
                        if (i >= n_x) continue;
                        const int k_at = (wide ? wide_at : x ? narrow_b : narrow_a) + i + 1;
                        const int k_st = wide ? k_at % KST : x * KSN + k_at % KSN;
                        const int v_st = wide ? (k_at - 1) % VSW : x * VSN + (k_at - 1) % VSN;
                        if (i >= 0) {
                            spin(&p_full[x], ((x ? done_b : done_a) + i) & 1);
                            if (!ok) break;
                            const uint64_t vd = v_desc + ((v_st * TILE) >> 4);          // O_x += P_x V
#pragma unroll
                            for (int k16 = 0; k16 < kTile / 16; ++k16)
                                t5::mma_ts(tmem_o + x * kTile, tmem_s + x * kTile + 8 * k16, vd + ((k16 * 16 * 128) >> 4), idesc_pv,
                                           (i > 0 || k16 > 0) ? 1u : 0u);
                        }
                        if (i + 1 < n_x) {
                            // the first tiles' arrival is tested here, the others' by the warp group that announces P
                            if (i < 0 && (x == 0 || !wide)) wait(&k_full[wide][k_st], (wide ? k_at / KST : k_at / KSN) & 1);
                            if (!ok) break;
                            const uint64_t kd = k_desc + ((k_st * TILE) >> 4);          // S_x = Q_x K^T
                            const uint64_t qd = q_desc + (wide && x ? (Q1 - Qs) >> 4 : 0);
#pragma unroll
                            for (int k16 = 0; k16 < HD / 16; ++k16)
                                t5::mma_ss(tmem_s + x * kTile, qd + (((k16 >> 2) * kHalf + (k16 & 3) * 32) >> 4),
                                           kd + (((k16 >> 2) * kHalf + (k16 & 3) * 32) >> 4), idesc_qk, k16 > 0 ? 1u : 0u);
                            t5::commit(smem_u32(&s_full[x]));
                        }
                        if (!wide || x == (nx1 > 0)) {                                  // the tiles' last reader
                            if (i >= 0) t5::commit(smem_u32(&v_empty[wide][v_st]));
                            if (i + 1 < n_x) t5::commit(smem_u32(&k_empty[wide][k_st]));
                        }
                    }
                }
                if (!ok) break;
                t5::commit(smem_u32(&o_done));
                done_a += nx0;
                done_b += nx1;
                if (wide) {
                    wide_at += nt;
                } else {
                    narrow_a += nx0;
                    narrow_b += nx1;
                }
            }
            if (!ok) failed_s = 1;                                    // the others run out of their bounded waits
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");
        // ---- softmax: a thread per row of a warp group
        const int x = warp >> 2, quarter = warp & 3;                  // quarter: the lanes this warp may access
        const int row = quarter * 32 + lane;
        const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t s_addr = tmem_s + x * kTile + lane_addr;
        const uint32_t o_addr = tmem_o + lane_addr;
        bool ok = true;
        // this warp's share of a piece's query rows into shared memory: on their way, and there
        auto load_queries = [&](const PieceNote& p) {
            const int rows_w = p.wide ? 32 : 16, r0 = p.wide ? quarter * 32 : warp * 16;
            unsigned char* to = p.wide && x ? Q1 : Qs;
            const int token0 = p.token0 + (p.wide ? x * per_tile : 0);
            const int live = min(p.token0 + p.tokens - token0, per_tile) * b.per;
            constexpr int CH = HD / 8;                                // 16-byte pieces of a row
            constexpr int AT_ONCE = 32 / CH;                          // rows of one instruction
            const int chunk = lane % CH;
            if (p.tiles > 0) {
                for (int r = r0 + lane / CH; r < min(r0 + rows_w, live); r += AT_ONCE) {
                    const int t = r / b.per;
                    cp_async_16(smem_u32(to + (chunk >> 3) * kHalf + r * 128 + (((chunk & 7) ^ (r & 7)) << 4)),
                                q + (token0 + t) * q_stride + static_cast<size_t>(p.kvh * b.per + r - t * b.per) * HD + chunk * 8, 16);
                }
                cp_async_commit();
            }
        };
        auto announce_queries = [&]() {
            cp_async_wait<0>();
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&q_full));
        };
        int wide_at = 0, narrow_at = 0, done = 0;
        // the eight warps go on, or stop, together: they meet at barriers
        auto together = [&](int n) {
            if (!ok) tail.softmax_failed[n & 1] = 1;
            asm volatile("bar.sync 1, 256;\n" ::: "memory");
            ok = tail.softmax_failed[n & 1] == 0;
        };
        ok = get_piece(0, ok);
        if (ok && ring[0].tiles >= 0) {
            load_queries(ring[0]);
            announce_queries();
        }
        together(1);
        for (int n = 0; ok; ++n) {
            const PieceNote& p = ring[n % kPieces];
            if (p.tiles < 0) break;
            const int wide = p.wide, nt = p.tiles;
            const int my_token = row / b.per + (wide ? x * per_tile : 0);         // of the piece
            const int live = min(p.tokens - (wide ? x * per_tile : 0), per_tile) * b.per;      // rows of the group
            const int n_x = wide ? (live > 0 ? nt : 0) : (x ? nt / 2 : (nt + 1) / 2);
            const bool idle = quarter * 32 >= live;                   // no row of this warp is one of the batch
            // keys [lo, lo + span) are seen by this row
            const int lo = p.key_lo, first_end = min(p.key_hi, p.pos0 + (wide ? x * per_tile : 0) + 1);
            const int span = min(p.key_hi, p.pos0 + my_token + 1) - lo;
            float m = -INFINITY, l = 0.f;                             // m: the reference maximum in use (log2 units)
            for (int i = 0; i < n_x; ++i) {
                const int kb = p.key0 + (wide ? i : 2 * i + x) * kTile;
                const int v_at = wide ? wide_at + i : narrow_at + i;
                const int v_st = wide ? v_at % VSW : x * VSN + v_at % VSN;
                unsigned long long* vf = &v_full[wide][v_st];
                const int v_par = (wide ? v_at / VSW : v_at / VSN) & 1;
                const bool edge = kb < lo || kb + kTile > p.key_hi;   // value rows that are none of the piece's
                if (quarter == 0 || edge) ok = mbar_wait(smem_u32(vf), v_par, ok ? 400000 : 1) && ok;
                // On behalf of the issuer: the next tile's keys, too, have arrived before P is announced.  A wait by parity
                // wants to know that the stage's phase before has completed, so where a ring has one stage it comes
                // behind this tile's scores (which were made of that phase's keys).
                auto next_keys = [&]() {
                    const int k_at = v_at + 1;
                    const int k_st = wide ? k_at % KST : x * KSN + k_at % KSN;
                    ok = mbar_wait(smem_u32(&k_full[wide][k_st]), (wide ? k_at / KST : k_at / KSN) & 1, ok ? 400000 : 1) && ok;
                };
                const bool keys_late = KSN == 1 && !wide;
                if (quarter == 0 && i + 1 < n_x && !keys_late) next_keys();
                if (edge) {
                    const int pos = kb + row;
                    if (pos < lo || pos >= p.key_hi) {
                        unsigned char* v = Vs + v_st * TILE + row * 128;
#pragma unroll
                        for (int h = 0; h < HALVES; ++h)
#pragma unroll
                            for (int c = 0; c < 8; ++c)
                                *reinterpret_cast<uint4*>(v + h * kHalf + ((c ^ (row & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async();
                }
                ok = mbar_wait(smem_u32(&s_full[x]), (done + i) & 1, ok ? 400000 : 1) && ok;
                __syncwarp();
                t5::fence_after();
                if (!idle) {
                    const bool inner = kb >= lo && kb + kTile <= first_end;       // every row sees all keys
                    uint32_t sv[128];
                    ld128(s_addr, sv);
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    if (inner) {
#pragma unroll
                        for (int j = 0; j < 128; j += 2)
                            mx[(j >> 1) & 3] = fmax3(mx[(j >> 1) & 3], __uint_as_float(sv[j]), __uint_as_float(sv[j + 1]));
                    } else {
                        const int d0 = kb - lo;
#pragma unroll
                        for (int j = 0; j < 128; ++j) {
                            const bool seen = static_cast<unsigned>(d0 + j) < static_cast<unsigned>(span);
                            const float v = seen ? __uint_as_float(sv[j]) : -INFINITY;
                            sv[j] = __float_as_uint(v);
                            mx[j & 3] = fmaxf(mx[j & 3], v);
                        }
                    }
                    const float tmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale_log2e;
                    // the old reference maximum serves on unless the new one is more than 2^8 above it
                    float alpha = 1.f;
                    bool rescale = false;
                    if (m == -INFINITY) {
                        m = tmax;
                    } else if (tmax > m + 8.0f) {
                        alpha = fast_exp2(m - tmax);
                        m = tmax;
                        rescale = true;
                    }
                    if (__any_sync(0xffffffffu, rescale)) {
                        // (the commit behind s_full covered the output products issued before)
#pragma unroll 1
                        for (int c = 0; c < HD / 16; ++c) {
                            __syncwarp();
                            float ov[16];
                            uint32_t ow[16];
                            ld16(o_addr + x * kTile + c * 16, ov);
#pragma unroll
                            for (int j = 0; j < 16; ++j) ow[j] = __float_as_uint(ov[j] * alpha);
                            t5::st16(o_addr + x * kTile + c * 16, ow);
                        }
                        t5::wait_st();
                        l *= alpha;
                    }
                    const float neg_m = m == -INFINITY ? 0.f : -m;
                    const uint64_t scale2 = pair_f32(scale_log2e, scale_log2e), neg_m2 = pair_f32(neg_m, neg_m);
                    uint64_t ps2[2] = {pair_f32(0.f, 0.f), pair_f32(0.f, 0.f)};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t pk[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            float a0, a1;
                            unpair_f32(fma_f32x2(pair_f32(__uint_as_float(sv[c * 32 + 2 * j]), __uint_as_float(sv[c * 32 + 2 * j + 1])),
                                                 scale2, neg_m2), a0, a1);
                            const float p0 = fast_exp2(a0), p1 = fast_exp2(a1);
                            ps2[j & 1] = add_f32x2(ps2[j & 1], pair_f32(p0, p1));
                            pk[j] = pack_bf16(p0, p1);
                        }
                        t5::st16(s_addr + c * 16, pk);
                    }
                    float s0, s1, s2, s3;
                    unpair_f32(ps2[0], s0, s1);
                    unpair_f32(ps2[1], s2, s3);
                    l += (s0 + s2) + (s1 + s3);
                    t5::wait_st();
                }
                if (quarter == 0 && i + 1 < n_x && keys_late) next_keys();
                t5::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&p_full[x]));
            }
            done += n_x;
            if (wide) wide_at += nt;
            else narrow_at += n_x;
            ok = mbar_wait(smem_u32(&o_done), n & 1, ok ? 400000 : 1) && ok;
            __syncwarp();
            t5::fence_after();
            // the next piece's queries are on their way while the first half of this one's outputs is written, and its first
            // scores are computed during the second
            ok = get_piece(n + 1, ok);
            bool queries = ok && ring[(n + 1) % kPieces].tiles >= 0;
            if (queries) load_queries(ring[(n + 1) % kPieces]);

            const int head = p.kvh * b.per + row % b.per, token = p.token0 + my_token;
            const bool mine = row < live;
            const size_t at = part_row(b, p.prefix != 0, p.first != 0, blockIdx.x, token, head,
                                       my_token * b.per + row % b.per);
            if (wide) {
                if (mine) parts.ml[at] = make_float2(m, l);
                if (n_x > 0 && !idle) {
#pragma unroll 1
                    for (int c = 0; c < HD / 32; ++c) {
                        // (the loads are the whole warp's: whatever a compiler makes of the condition below, it meets here)
                        __syncwarp();
                        if (c == HD / 64 && queries) {
                            announce_queries();
                            queries = false;
                        }
                        float v[32];
                        t5::ld32(o_addr + x * kTile + c * 32, v);
                        if (mine) {
                            float* to = parts.o + at * HD + c * 32;
#pragma unroll
                            for (int d = 0; d < 32; d += 8) store8(to + d, v + d);
                        }
                    }
                }
            } else {
                // the two warp groups' outputs joined, half of the columns by each
                if (x == 0) tail.a_top[row] = m;
                else tail.b_state[row] = make_float2(m, l);
                asm volatile("bar.sync 1, 256;\n" ::: "memory");
                const float a_top = tail.a_top[row];
                const float2 bs = tail.b_state[row];
                const float top = fmaxf(a_top, bs.x);
                const float ca = a_top == -INFINITY ? 0.f : fast_exp2(a_top - top), cb = bs.x == -INFINITY ? 0.f : fast_exp2(bs.x - top);
                if (mine && x == 0) parts.ml[at] = make_float2(top, l * ca + bs.y * cb);
                if (nt > 0 && !idle) {
#pragma unroll 1
                    for (int c = 0; c < HD / 32; ++c) {
                        const uint32_t col = x * (HD / 2) + c * 16;
                        __syncwarp();
                        if (c == HD / 64 && queries) {
                            announce_queries();
                            queries = false;
                        }
                        float y[16];
                        ld16(o_addr + col, y);
#pragma unroll
                        for (int d = 0; d < 16; ++d) y[d] *= ca;
                        if (nt > 1) {
                            float v[16];
                            ld16(o_addr + kTile + col, v);
#pragma unroll
                            for (int d = 0; d < 16; ++d) y[d] = fmaf(v[d], cb, y[d]);
                        }
                        if (mine) {
                            store8(parts.o + at * HD + col, y);
                            store8(parts.o + at * HD + col + 8, y + 8);
                        }
                    }
                }
            }
            if (queries) announce_queries();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&piece_empty[n % kPieces]));
            t5::fence_before();
            together(n);                                              // (and the other group's outputs have been read)
            t5::fence_after();
        }
        if (!ok) failed_s = 1;
    }
    t5::fence_before();
    __syncthreads();
    if (warp == 9) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base_s), "r"(TmemCols) : "memory");
    }
    if (tid == 0 && failed_s) atomicExch(&g_shared_error, 1);
}

template <int HD>
static int launch_tc(const CUtensorMap& k_map, const CUtensorMap& v_map, const Batch& b, const void* q, long long q_stride,
                     float scale, Note* notes, unsigned* header, Parts parts, int ctas, cudaStream_t stream) {
    allow_smem<shared_attention_tc_kernel<HD>>(tc_smem(HD));
    return launch_pdl(shared_attention_tc_kernel<HD>, dim3(ctas), dim3(kTcThreads), tc_smem(HD), stream, k_map, v_map, b,
                      static_cast<const __nv_bfloat16*>(q), q_stride, scale * 1.4426950408889634f, notes, header, parts);
}

int shared_attention_tc(Batch b, const void* q, long long q_stride, const void* keys, const void* values, int hd, float scale,
                        Note* notes, unsigned* header, Parts parts, int ctas, cudaStream_t stream) {
    const long long rows = static_cast<long long>(b.num_pages) * b.nkv * b.page_size;
    if (!somi_shared_attention_tc_takes(b.nq, b.nkv, hd, b.page_size) || rows > 0x7fffffffll) return SOMI_ERR_UNSUPPORTED;
    // (made in every call: nothing is kept by an address)
    alignas(64) CUtensorMap k_map, v_map;
    if (make_tensor_map_bf16_2d(&k_map, keys, rows, hd, b.page_size, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
        make_tensor_map_bf16_2d(&v_map, values, rows, hd, b.page_size, 64, CU_TENSOR_MAP_SWIZZLE_128B))
        return SOMI_ERR_UNSUPPORTED;
    b.wide_tokens = kTile / b.per;
    b.item_tokens = 2 * b.wide_tokens;
    b.align = b.unit_wide = kTile;
    b.unit_narrow = 2 * kTile;
    b.over_wide = kOverWide;
    return hd == 64 ? launch_tc<64>(k_map, v_map, b, q, q_stride, scale, notes, header, parts, ctas, stream)
                    : launch_tc<128>(k_map, v_map, b, q, q_stride, scale, notes, header, parts, ctas, stream);
}

}  // namespace shp
}  // namespace somi

using namespace somi;

SOMI_API int somi_shared_attention_tc_takes(int nq, int nkv, int hd, int page_size) {
    return nkv > 0 && nq % nkv == 0 && nq / nkv <= shp::kTile && (hd == 64 || hd == 128) && page_size >= 8 &&
           shp::kTile % page_size == 0;
}
SOMI_API int somi_shared_attention_tc_block_rows() { return shp::kTcBlockRows; }
SOMI_API int somi_shared_attention_error() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, shp::g_shared_error, sizeof(int)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(shp::g_shared_error, &zero, sizeof(int));
    return v;
}
