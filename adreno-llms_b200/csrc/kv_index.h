// Index arithmetic of the paged key/value cache, shared by its kernels and the host (plain C++: it is also tested without a GPU).
//
// Pages are [page][kv head][slot][dim], their scales [page][kv head][slot]; a page holds 1 << page_shift positions.  All that a
// kernel takes from device memory (row starts, lengths, page numbers) goes through the checks here before it becomes an address.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define NNB_HD __host__ __device__ __forceinline__
#else
#define NNB_HD inline
#endif

namespace nnb {

enum KvFmt : int { KV_FP16 = 0, KV_INT8 = 1, KV_FP8 = 2 };
NNB_HD constexpr int kv_cell_bytes(int fmt) { return fmt == KV_FP16 ? 2 : 1; }
NNB_HD constexpr float kv_max_code(int fmt) { return fmt == KV_INT8 ? 127.f : 448.f; }

// The new rows of a sequence and its length, brought into range: 0 <= row0 <= row1 <= num_rows, 0 <= len <= max_len.
struct SeqExtent {
    int row0, row1, len;
    bool bad;   // something had to be cut
};
NNB_HD SeqExtent seq_extent(int start, int end, int kv_len, int num_rows, int max_len) {
    SeqExtent e;
    e.row0 = start < 0 ? 0 : start > num_rows ? num_rows : start;
    e.row1 = end < e.row0 ? e.row0 : end > num_rows ? num_rows : end;
    e.bad = start < 0 || end < start || end > num_rows || kv_len < 0 || kv_len > max_len;
    e.len = kv_len < 0 ? 0 : kv_len > max_len ? max_len : kv_len;
    return e;
}

NNB_HD bool page_ok(int page, int num_pages) { return page >= 0 && page < num_pages; }

// The row of a cell among all rows of the pages ([page][kv head][slot]); 64 bits, for a cache passes 2^31 values.
NNB_HD int64_t cell_row(int page, int head, int slot, int kv_heads, int page_shift) {
    return (((int64_t)page * kv_heads + head) << page_shift) + slot;
}

// Keys that the query at position p sees: [lo, p] and [0, min(sinks, lo)).  Without a window lo is 0.  p < 0: none.
NNB_HD int window_begin(int p, int window) { return window > 0 && p >= window ? p - window + 1 : 0; }
NNB_HD bool key_visible(int key, int p, int window, int sinks) { return key <= p && (key >= window_begin(p, window) || key < sinks); }

// The tiles of `tile` keys that some query with a position in [p0, p1] sees, counted from key 0: first those with sinks, then those from
// the window of p0 to p1.  tile_at(i), 0 <= i < tiles(), walks them in order.
struct TileRange {
    int sink_tiles, first, end;
    NNB_HD int tiles() const { return sink_tiles + end - first; }
    NNB_HD int tile_at(int i) const { return i < sink_tiles ? i : first + (i - sink_tiles); }
};
NNB_HD TileRange visible_tiles(int p0, int p1, int window, int sinks, int tile) {
    TileRange r;
    if (p1 < 0) {
        r.sink_tiles = r.first = r.end = 0;
        return r;
    }
    r.first = window_begin(p0 < 0 ? 0 : p0, window) / tile;
    r.end = p1 / tile + 1;
    const int s = window > 0 && sinks > 0 ? (sinks - 1) / tile + 1 : 0;   // (1 <= sinks: no overflow)
    r.sink_tiles = s < r.first ? s : r.first;
    return r;
}

}  // namespace nnb
