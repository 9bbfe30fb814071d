// How a call's work is dealt out to blocks.
//
// An item is a tile of queries (up to `tokens` new tokens of one sequence, times the `group` query heads that share a cache head) with the
// key tiles that some of them see, at least one (an item that sees nothing still has zeros to write).  Items are numbered by
// sequence, head and query tile, their key tiles are strung together, and block b takes units [b * chunk, (b + 1) * chunk) of that string:
// every block has the same number, whatever the lengths are, and all lengths stay on the device, so that a recorded call takes new ones.
// A piece of an item in one block is a segment; the blocks of an item that is cut leave partial results to be joined.
// An item also costs its block something that does not depend on its keys (queries to fetch, sums to write): `extra` units in front of its
// first key tile stand for that.  (Without them a causal prompt's first query tiles, of few keys, came ten to a block: 4096 tokens of 32 heads of 64 dims
// in fp16 had blocks of 190 and of 317 thousand clocks.)
// Where there are at least twice as many blocks as items, each item is filled up to whole chunks, so that no block has parts of two: it would only
// have two segments to finish, one after the other (with / without, us: a token to 700 positions of 3 heads of 64 dims, int8, 9.3 / 16.6; two tokens each
// of 8 sequences of 300 positions, 8 heads of 128 dims, e4m3, 7.9 / 16.8).
#pragma once
#include "kv_cells.cuh"

namespace nnb {

struct WorkShape {
    int group;     // query heads of a token in an item
    int tokens;    // tokens of an item
    int vheads;    // items side by side: cache heads (times the parts of a head's query heads)
    int tile;      // keys of a unit
    int window, sinks;
    unsigned extra;   // units of an item besides its key tiles
    unsigned chunk;   // units of a block, and whether items are filled up to it
    bool pad;
    __device__ __forceinline__ unsigned units(unsigned tiles) const { return pad ? (tiles + chunk - 1) / chunk * chunk : tiles + extra; }
};

struct SeqWork {
    int row0, n, len, tiles_q;   // first row, new tokens, length, query tiles
};

struct Segment {
    int seq, vhead, qt;
    int row0, n, len;       // of the sequence
    int first, count;       // key tiles [first, first + count) of the item
    int total;              // key tiles of the item
    unsigned unit0;         // number of the item's first key tile
    // positions of the item's first and last token
    __device__ __forceinline__ int p0(const WorkShape& w) const { return len - n + qt * w.tokens; }
    __device__ __forceinline__ int p1(const WorkShape& w) const { return len - n + min((qt + 1) * w.tokens, n) - 1; }
    __device__ __forceinline__ TileRange tiles(const WorkShape& w) const { return visible_tiles(p0(w), p1(w), w.window, w.sinks, w.tile); }
};

__device__ __forceinline__ SeqWork load_seq(const KvSeqs& s, const WorkShape& w, int i, bool* bad = nullptr, bool* descends = nullptr) {
    const int start = s.row_start[i], end = s.row_start[i + 1];
    const SeqExtent e = seq_extent(start, end, s.kv_len[i], s.num_rows, s.max_len);
    if (bad) *bad = e.bad;
    if (descends) *descends = end < start;
    SeqWork q;
    q.row0 = e.row0;
    q.n = e.row1 - e.row0;
    q.len = e.len;
    q.tiles_q = q.n <= w.tokens ? (q.n > 0) : (q.n + w.tokens - 1) / w.tokens;   // (a division costs as much as a load from the L2)
    return q;
}
__device__ __forceinline__ int item_tiles(const SeqWork& q, const WorkShape& w, int qt) {
    const int p0 = q.len - q.n + qt * w.tokens, p1 = q.len - q.n + min((qt + 1) * w.tokens, q.n) - 1;
    return max(1, visible_tiles(p0, p1, w.window, w.sinks, w.tile).tiles());
}
// Units of all query tiles of a sequence; by each lane for one of its own.  (Where some lane's sequence has many, the warp goes through them
// together.)
__device__ __forceinline__ unsigned seq_tiles(const SeqWork& q, const WorkShape& w) {
    const int lane = threadIdx.x & 31;
    unsigned t = 0;
    const bool deep = q.tiles_q > 4;
    if (!deep)
        for (int i = 0; i < q.tiles_q; ++i) t += w.units(item_tiles(q, w, i));
    for (unsigned left = __ballot_sync(0xffffffffu, deep); left; left &= left - 1) {
        const int from = __ffs(left) - 1;
        SeqWork o;
        o.row0 = 0;
        o.n = __shfl_sync(0xffffffffu, q.n, from);
        o.len = __shfl_sync(0xffffffffu, q.len, from);
        o.tiles_q = __shfl_sync(0xffffffffu, q.tiles_q, from);
        unsigned x = 0;
        for (int i = lane; i < o.tiles_q; i += 32) x += w.units(item_tiles(o, w, i));
        x = __reduce_add_sync(0xffffffffu, x);
        if (lane == from) t = x;
    }
    return t;
}

// Where a block's units are.  Copies of a walk go on independently; next() is called by whole warps.
struct Walk {
    unsigned u, end;      // the next unit, and the block's last one + 1
    int seq, vhead, qt, first;
    SeqWork q;

    __device__ __forceinline__ bool next(const KvSeqs& s, const WorkShape& w, Segment* out) {
        if (u >= end) return false;
        while (qt >= q.tiles_q) {
            qt = 0;
            if (q.tiles_q == 0 || ++vhead >= w.vheads) {
                vhead = 0;
                if (++seq >= s.num_seqs) {   // (no units are left: not reached while u < end)
                    u = end;
                    return false;
                }
                q = load_seq(s, w, seq);
            }
        }
        const int total = item_tiles(q, w, qt);
        if (!w.pad) {   // (`first` counts from the item's first unit: only the key tiles are worked on)
            const unsigned skip = first < (int)w.extra ? min(w.extra - first, end - u) : 0u;
            u += skip;
            first += skip;
            if (u >= end) return false;
            first -= w.extra;
        }
        out->seq = seq;
        out->vhead = vhead;
        out->qt = qt;
        out->row0 = q.row0;
        out->n = q.n;
        out->len = q.len;
        out->first = first;
        out->total = total;
        out->unit0 = u - first;
        out->count = (int)min((unsigned)(total - first), end - u);
        u = w.pad ? end : u + out->count;
        first = 0;
        ++qt;
        return true;
    }
};

// The walk of this block, found by each warp for itself: the sequences, one per lane, how many units there are and where this block's begin.
// `least`: the fewest units that are worth a block (a unit for each warp of the kernel for few rows, against 1: a token to 2048 positions of 2 heads of 64
// dims, fp16, 8.5 / 11.0 us).  w->chunk and w->pad are set.
// The host has seen to it that units are fewer than 2^31 as long as no row belongs to two sequences: row starts that do not ascend are no work at all.
__device__ __forceinline__ Walk find_work(const KvSeqs& s, WorkShape* w, unsigned least, int* status) {
    const int lane = threadIdx.x & 31;
    Walk k;
    k.u = k.end = 0;
    k.seq = k.vhead = k.qt = k.first = 0;
    k.q = SeqWork{0, 0, 0, 0};
    SeqWork q = k.q;
    unsigned total = 0, items = 0;
    const unsigned extra = w->extra;
    w->extra = 0;
    w->pad = false;
    w->chunk = 1;
    bool disorder = false;
    auto load = [&](int i0) {
        bool bad = false, descends = false;
        q = SeqWork{0, 0, 0, 0};
        if (i0 + lane < s.num_seqs) q = load_seq(s, *w, i0 + lane, &bad, &descends);
        if (bad) status[STATUS_BAD_TABLE] = 1;
        disorder |= descends;
    };
    unsigned tiles = 0;
    for (int i0 = 0; i0 < s.num_seqs; i0 += 32) {
        load(i0);
        tiles = seq_tiles(q, *w);
        total += __reduce_add_sync(0xffffffffu, tiles);
        items += __reduce_add_sync(0xffffffffu, (unsigned)q.tiles_q);
    }
    if (__any_sync(0xffffffffu, disorder)) return k;
    total *= w->vheads;
    items *= w->vheads;
    w->pad = 2 * items <= gridDim.x;
    const unsigned blocks = w->pad ? gridDim.x - items : gridDim.x;   // (filled up, items take up to one more block each)
    if (!w->pad) {
        w->extra = extra;
        total += items * extra;
    }
    w->chunk = max(least, (total + blocks - 1) / blocks);
    k.u = blockIdx.x * w->chunk;
    unsigned base = 0;
    for (int i0 = 0; i0 < s.num_seqs; i0 += 32) {
        if (s.num_seqs > 32) load(i0);
        // (of a head; what has been counted above serves where items are not filled up, or are one to a sequence)
        const unsigned head = s.num_seqs <= 32 && !w->pad                                             ? tiles + q.tiles_q * w->extra
                              : s.num_seqs <= 32 && __all_sync(0xffffffffu, q.tiles_q <= 1) ? (q.tiles_q ? w->units(tiles) : 0u)
                                                                                            : seq_tiles(q, *w);
        const unsigned mine = head * w->vheads;
        unsigned upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, base + upto > k.u);
        if (!hit) {
            base += __shfl_sync(0xffffffffu, upto, 31);
            continue;
        }
        const int l = __ffs(hit) - 1;   // the sequence of the block's first unit
        unsigned rest = k.u - base - __shfl_sync(0xffffffffu, upto - mine, l);
        const unsigned per_head = __shfl_sync(0xffffffffu, head, l);
        k.seq = i0 + l;
        k.q.row0 = __shfl_sync(0xffffffffu, q.row0, l);
        k.q.n = __shfl_sync(0xffffffffu, q.n, l);
        k.q.len = __shfl_sync(0xffffffffu, q.len, l);
        k.q.tiles_q = __shfl_sync(0xffffffffu, q.tiles_q, l);
        k.vhead = (int)(rest / per_head);
        rest -= k.vhead * per_head;
        if (k.q.tiles_q > 1) {
            for (int q0 = 0;; q0 += 32) {   // and its query tile
                const unsigned n = q0 + lane < k.q.tiles_q ? w->units(item_tiles(k.q, *w, q0 + lane)) : 0u;
                unsigned run = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned x = __shfl_up_sync(0xffffffffu, run, o);
                    if (lane >= o) run += x;
                }
                const unsigned in = __ballot_sync(0xffffffffu, run > rest);
                if (in || q0 + 32 >= k.q.tiles_q) {
                    const int j = in ? __ffs(in) - 1 : 0;
                    k.qt = q0 + j;
                    rest -= __shfl_sync(0xffffffffu, run - n, j);
                    break;
                }
                rest -= __shfl_sync(0xffffffffu, run, 31);
            }
        }
        k.first = (int)rest;
        k.end = w->pad ? k.u + w->chunk : min(total, k.u + w->chunk);
        return k;
    }
    k.u = k.end = 0;   // no units for this block
    return k;
}

}  // namespace nnb
