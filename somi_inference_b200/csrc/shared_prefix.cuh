// Attention of a batch whose requests share their first positions in groups: how the work of a call is
// cut, and how its parts are joined.  Used by the kernels of attention_shared.cu (any size) and
// attention_shared_tcgen05.cu (tensor cores).
//
// An *entry* is a set of query rows that read the same keys: the tokens of a whole group over the
// group's prefix, or the tokens of one request over its own positions behind the prefix.  Entries
// 0 .. G-1 are the groups, G .. G+R-1 the requests.  An entry's tokens are cut into tiles of
// `item_tokens`; a tile for one key/value head is an *item*, its rows are the tile's tokens times the
// query heads of that head, and its keys are cut into *units*.  An item costs its units and one unit
// more, or `over_wide` (queries to be gathered, rows to be written), and the costs of all items, one behind the other, are shared out evenly over the CTAs in
// contiguous ranges (U / N costs each, the first U % N of them one more).  So any mixture of long and
// short entries fills the chip evenly, whatever the lengths are, and the host has to know none of them
// (a captured graph runs with new lengths).  Every CTA adds the entries' costs up by itself (a few loads and one scan over the
// block), which takes less time than a kernel in front that writes them down.
//
// A piece of an item that a CTA computes leaves its rows' output (not divided by its sum), their maximum and their sum.  Only
// the first piece of a CTA's range can be the continuation of an item that another CTA began, so the
// partial results lie in three regions: the first pieces of prefixes, one row per (token, head); the first pieces of
// the requests' own keys, likewise; and one block of rows for each CTA's continuation.  `shared_merge_kernel` joins them:
// m = max m_i, l = sum l_i 2^(m_i - m), out = sum o_i 2^(m_i - m) / l  (float32, base 2).
#pragma once

#include "common.cuh"

namespace somi {
namespace shp {

constexpr int kMaxEntries = 8192;   // groups and requests of a call
constexpr int kOwned = 64;          // entries whose tokens one CTA notes for the merge, at most
constexpr int kFewRows = 16;        // query rows of an entry that attention_shared_rows.cu takes

struct Batch {
    const int *cu_q;                // [R + 1], or null: one token per request
    const int *ctx_len, *prefix_len, *group_off, *block_table;
    int bt_stride, R, G, T, nq, nkv, per, page_size, num_pages;
    int item_tokens;                // tokens of a tile, at most
    int wide_tokens;                // entries of more tokens than this have units of `unit_wide` keys
    int unit_narrow, unit_wide, align;       // keys; powers of two
    int over_wide;                  // what their items cost beside their units (others: 1)
    int block_rows;                 // rows of a CTA's continuation
};

// The groups' borders and prefixes as a block reads them: its own copies where they are few; else the step's arrays, which are
// read before the kernels in front have ended, and so through L2.
struct Groups {
    const int *off, *prefix;
    bool held;
    __device__ __forceinline__ int border(int g) const { return held ? off[g] : ld_step(off + g); }
    __device__ __forceinline__ int shared(int g) const { return held ? prefix[g] : ld_step(prefix + g); }
};

// What joins the parts: per token, for the prefix and for its own keys, where the item of its first
// key/value head begins in the order of costs, what an item costs, how many units it has, and the
// token's place in the tile (with a flag).
struct Note { unsigned begin; int cost, units, place; };
constexpr int kHasPrefix = 1 << 30;

struct Entry {
    int first, tokens;              // rows of the batch
    int table;                      // the request whose block table leads to the keys
    int key_lo, key_hi;             // keys [key_lo, key_hi)
    int pos0;                       // position of the first token: token i sees keys up to pos0 + i
    int tiles, unit, units;         // tiles of tokens, keys of a unit, units of an item
    int over;                       // what an item costs beside its units
    __device__ __forceinline__ int cost() const { return units + over; }
    __device__ __forceinline__ int base(const Batch& b) const { return key_lo & -b.align; }
};

__device__ __forceinline__ int clamped(int x, int lo, int hi) { return min(max(x, lo), hi); }

__device__ __forceinline__ int token_of(const Batch& b, int r) {
    return b.cu_q ? clamped(ld_step(b.cu_q + r), 0, b.T) : r;
}

// The group that request r is in, or -1.  (Groups are runs of neighbouring requests.)
__device__ __forceinline__ int group_of(const Batch& b, const Groups& g, int r) {
    int lo = 0, hi = b.G;           // the last group that begins at or in front of r
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (g.border(mid) <= r) lo = mid + 1;
        else hi = mid;
    }
    return lo > 0 && r < g.border(lo) ? lo - 1 : -1;
}

// What the arrays say about a request.
struct Raw { int ctx, first, end; };
__device__ __forceinline__ Raw raw_of(const Batch& b, int r) {
    return Raw{ld_step(b.ctx_len + r), token_of(b, r), b.cu_q ? token_of(b, r + 1) : r + 1};
}

// Everything that lengths lead to stays inside the batch's rows and the table's columns, whatever they hold.  `raw`: of a request's entry.
__device__ __forceinline__ Entry entry_of(const Batch& b, const Groups& gs, int e, const Raw& raw) {
    Entry x;
    const int span = b.bt_stride * b.page_size;
    if (e < b.G) {
        const int r0 = clamped(gs.border(e), 0, b.R), r1 = clamped(gs.border(e + 1), r0, b.R);
        x.table = min(r0, b.R - 1);
        x.first = token_of(b, r0);
        x.tokens = r1 > r0 ? max(token_of(b, r1) - x.first, 0) : 0;
        x.key_lo = 0;
        x.key_hi = clamped(gs.shared(e), 0, span);
        x.pos0 = 0x3fffffff;        // every token sees the whole prefix
    } else {
        const int r = e - b.G, g = group_of(b, gs, r);
        x.table = r;
        x.first = raw.first;
        x.tokens = max(raw.end - x.first, 0);
        const int ctx = clamped(raw.ctx, 0, span);
        x.key_lo = g >= 0 ? clamped(gs.shared(g), 0, ctx) : 0;
        x.key_hi = min(ctx + x.tokens, span);
        x.pos0 = ctx;
    }
    const bool wide = x.tokens > b.wide_tokens;
    x.unit = wide ? b.unit_wide : b.unit_narrow;
    x.over = wide ? b.over_wide : 1;
    const bool some = x.tokens > 0 && x.key_hi > x.key_lo;
    x.tiles = some ? (x.tokens + b.item_tokens - 1) / b.item_tokens : 0;
    x.units = some ? (x.key_hi - x.base(b) + x.unit - 1) >> (31 - __clz(x.unit)) : 0;
    return x;
}
__device__ __forceinline__ Entry entry_of(const Batch& b, const Groups& gs, int e) {
    return entry_of(b, gs, e, e >= b.G ? raw_of(b, e - b.G) : Raw{0, 0, 0});
}

// How `total` costs are shared out over `n` CTAs.
struct Shares {
    unsigned each, more;            // the first `more` CTAs take each + 1
    __device__ __forceinline__ Shares(unsigned total, unsigned n) : each(total / n), more(total % n) {}
    __device__ __forceinline__ unsigned begin(unsigned b) const { return b * each + min(b, more); }
    __device__ __forceinline__ unsigned cta_of(unsigned cost) const {
        const unsigned wide = more * (each + 1);
        return cost < wide ? cost / (each + 1) : more + (cost - wide) / each;     // (each = 0: cost < wide)
    }
};

// A CTA's range of costs.
struct Range {
    unsigned total;                 // all costs
    unsigned begin, end;            // this CTA's
    int entry;                      // the entry that holds `begin`
    unsigned entry_base;            // where that entry begins
    Entry at;                       // that entry
};

struct RangeScratch {
    unsigned warp_sum[32];
    int entry;
    unsigned entry_base;
    Entry at;                       // that entry
};

constexpr int kGroupsHeld = 31;     // groups that a block copies
struct GroupScratch {
    int off[kGroupsHeld + 1], prefix[kGroupsHeld + 1];
};

// All threads of the block, first of all.  `raw`: what find_range asks for next, so that it is on its way meanwhile.
template <int THREADS>
__device__ __forceinline__ Groups hold_groups(const Batch& b, GroupScratch& s, Raw& raw) {
    const int i = threadIdx.x, r = i * ((b.G + b.R + THREADS - 1) / THREADS) - b.G;
    raw = r >= 0 && r < b.R ? raw_of(b, r) : Raw{0, 0, 0};
    if (b.G > kGroupsHeld) return Groups{b.group_off, b.prefix_len, false};
    if (i <= b.G) s.off[i] = ld_step(b.group_off + i);
    if (i >= 32 && i - 32 < b.G) s.prefix[i - 32] = ld_step(b.prefix_len + i - 32);
    __syncthreads();
    return Groups{s.off, s.prefix, true};
}

// All threads of the block.  owned[k]: where entry blockIdx.x + k gridDim.x begins, whose tokens this CTA notes.
template <int THREADS>
__device__ __forceinline__ Range find_range(const Batch& b, const Groups& gs, const Raw& raw, RangeScratch& s, unsigned* owned) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int E = b.G + b.R, each = (E + THREADS - 1) / THREADS;
    const int e0 = tid * each, e1 = min(e0 + each, E);
    unsigned mine = 0;
    Entry first_entry;
    for (int e = e0; e < e1; ++e) {
        const Entry x = e == e0 ? entry_of(b, gs, e, raw) : entry_of(b, gs, e);
        if (e == e0) first_entry = x;
        mine += static_cast<unsigned>(x.tiles) * x.cost() * b.nkv;
    }
    unsigned incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned n = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += n;
    }
    if (lane == 31) s.warp_sum[warp] = incl;
    if (tid == 0) s.entry = -1;
    __syncthreads();
    unsigned before = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        const unsigned v = s.warp_sum[w];
        if (w < warp) before += v;
        total += v;
    }
    Range r;
    r.total = total;
    const Shares shares(total, gridDim.x);
    r.begin = shares.begin(blockIdx.x);
    r.end = shares.begin(blockIdx.x + 1);
    const bool holds = r.begin >= before && r.begin < before + mine;
    unsigned at = before;
    for (int e = e0; e < e1; ++e) {
        const Entry x = e == e0 ? first_entry : entry_of(b, gs, e);
        const unsigned c = static_cast<unsigned>(x.tiles) * x.cost() * b.nkv;
        if (holds && r.begin >= at && r.begin < at + c) {
            s.entry = e;
            s.entry_base = at;
            s.at = x;
        }
        if (e % gridDim.x == blockIdx.x) owned[e / gridDim.x] = at;
        at += c;
    }
    __syncthreads();
    r.entry = s.entry;
    r.entry_base = s.entry_base;
    r.at = s.at;
    return r;
}

// The notes of this CTA's entries.  `notes`: [2][T], prefixes first; header[0]: all costs.  After the wait for the kernels
// in front.
template <int THREADS>
__device__ __forceinline__ void write_notes(const Batch& b, const Groups& gs, const unsigned* owned, unsigned total, Note* notes,
                                            unsigned* header, int thread) {
    if (blockIdx.x == 0 && thread == 0) header[0] = total;
    for (int e = blockIdx.x, k = 0; e < b.G + b.R; e += gridDim.x, ++k) {
        const Entry x = entry_of(b, gs, e);
        if (e < b.G && x.tiles == 0) continue;      // (the requests' own notes say whether there is a prefix)
        Note* to = notes + (e < b.G ? 0 : b.T) + x.first;
        for (int t = thread; t < x.tokens; t += THREADS) {
            Note n;
            const int j = t / b.item_tokens;
            n.begin = owned[k] + static_cast<unsigned>(j) * x.cost() * b.nkv;
            n.cost = x.cost();
            n.units = x.units;
            n.place = t - j * b.item_tokens;
            if (e >= b.G && x.key_lo > 0) n.place |= kHasPrefix;
            if (x.tiles == 0) n.units = 0;
            to[t] = n;
        }
    }
}

// A CTA's pieces, one after the other.
struct Piece {
    Entry x;
    int tile, kvh;
    int unit0, unit1;               // units [unit0, unit1) of the item
    bool first;                     // the item begins in this CTA
    int tokens;                     // of the tile
    int token0;                     // its first row of the batch
};

struct Walk {
    unsigned at, end;               // costs
    int e;
    unsigned base;
    Entry x;
    __device__ __forceinline__ Walk(const Range& r) : at(r.begin), end(r.end), e(r.entry), base(r.entry_base), x(r.at) {}
    __device__ __forceinline__ bool next(const Batch& b, const Groups& gs, Piece& p) {
        while (at < end) {
            unsigned whole = static_cast<unsigned>(x.tiles) * x.cost() * b.nkv;
            while (at >= base + whole) {            // (the range ends inside an entry, so this ends)
                base += whole;
                if (++e >= b.G + b.R) return false;
                x = entry_of(b, gs, e);
                whole = static_cast<unsigned>(x.tiles) * x.cost() * b.nkv;
            }
            const unsigned cost = x.cost();
            const unsigned item = (at - base) / cost, o = (at - base) - item * cost;
            const unsigned stop = min(end - at + o, cost);
            at += stop - o;
            const unsigned over = x.over;
            p.unit0 = o > over ? o - over : 0;
            p.unit1 = stop > over ? stop - over : 0;
            p.tile = item / b.nkv;
            p.kvh = item % b.nkv;
            p.first = o == 0;
            p.token0 = x.first + p.tile * b.item_tokens;
            p.tokens = min(b.item_tokens, x.tokens - p.tile * b.item_tokens);
            if (p.unit1 > p.unit0) {
                p.x = x;
                return true;
            }
        }
        return false;
    }
};

// Where the rows of a piece go.  Rows of first pieces: (token, head), of prefixes and of own keys; of continuations: the CTA's block.
struct Parts {
    float* o;                       // [rows, hd]
    float2* ml;                     // [rows]
};
__device__ __forceinline__ size_t part_row(const Batch& b, bool prefix, bool first, int cta, int token, int head, int row_in_item) {
    if (first) return ((prefix ? 0 : static_cast<size_t>(b.T)) + token) * b.nq + head;
    return 2 * static_cast<size_t>(b.T) * b.nq + static_cast<size_t>(cta) * b.block_rows + row_in_item;
}

// The kernels on tensor cores, for calls of few rows (attention_shared_rows.cu) and for any (attention_shared_tcgen05.cu):
// they set their own sizes of tiles in `b`.
int shared_attention_rows(Batch b, const void* q, long long q_stride, const void* keys, const void* values, int hd, float scale,
                          Note* notes, unsigned* header, Parts parts, int ctas, cudaStream_t stream);
int shared_attention_tc(Batch b, const void* q, long long q_stride, const void* keys, const void* values, int hd, float scale,
                        Note* notes, unsigned* header, Parts parts, int ctas, cudaStream_t stream);

}  // namespace shp
}  // namespace somi

SOMI_API int somi_shared_attention_tc_takes(int nq, int nkv, int hd, int page_size);
SOMI_API int somi_shared_attention_tc_block_rows();
