// What the C-ABI calls on a key/value cache share: the handle, and checks of arguments.
#pragma once
#include <cuda_runtime.h>

#include "../../include/nnopt_b200.h"
#include "attention.h"
#include "attention_maps.h"
#include "internal.h"

struct nn_kv_cache {
    int device;
    nnb::KvView view;
    nnb::AttnMaps maps;
};

namespace nnb {

inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

inline size_t cache_bytes(const KvView& v) {
    return ((size_t)v.num_pages * v.kv_heads << v.page_shift) * (size_t)v.dim * kv_cell_bytes(v.fmt);
}

// Rows of `width` values at a distance of `stride`.
struct Rows {
    const uint16_t* p;
    int64_t stride, width;
};
inline size_t rows_bytes(const Rows& r, int rows) { return ((size_t)(rows - 1) * r.stride + r.width) * 2; }

// Whether two sets of rows share memory.  Of equal stride they may be columns of one buffer (q, k and v of a fused projection).
inline bool rows_overlap(const Rows& a, const Rows& b, int rows) {
    const char *pa = (const char*)a.p, *pb = (const char*)b.p;
    if (pa >= pb + rows_bytes(b, rows) || pb >= pa + rows_bytes(a, rows)) return false;
    if (a.stride != b.stride) return true;
    const int64_t pitch = a.stride * 2;
    int64_t d = (int64_t)((intptr_t)pb - (intptr_t)pa) % pitch;
    if (d < 0) d += pitch;
    return d < a.width * 2 || d + b.width * 2 > pitch;
}
inline bool share(const void* p, size_t np, const void* q, size_t nq) { return p && q && (const char*)p < (const char*)q + nq && (const char*)q < (const char*)p + np; }
inline size_t scale_bytes(const KvView& v) { return cache_bytes(v) / ((size_t)v.dim * kv_cell_bytes(v.fmt)) * 2; }
inline bool over_cache(const void* p, size_t n, const KvView& v) {
    const size_t nc = cache_bytes(v), ns = scale_bytes(v);
    return share(p, n, v.k, nc) || share(p, n, v.v, nc) || share(p, n, v.k_scale, ns) || share(p, n, v.v_scale, ns);
}
inline bool rows_over_cache(const Rows& r, int rows, const KvView& v) { return over_cache(r.p, rows_bytes(r, rows), v); }
// (what a call writes must not be what tells it where to)
inline bool cache_over_batch(const KvView& v, const nn_kv_batch* b) {
    return over_cache(b->row_start, 4 * ((size_t)b->num_seqs + 1), v) || over_cache(b->kv_len, 4 * (size_t)b->num_seqs, v) ||
           over_cache(b->page_table, 4 * (size_t)b->num_seqs * b->table_stride, v);
}
inline bool rows_over_batch(const Rows& r, const nn_kv_batch* b) {
    const size_t n = rows_bytes(r, b->num_rows);
    return share(r.p, n, b->row_start, 4 * ((size_t)b->num_seqs + 1)) || share(r.p, n, b->kv_len, 4 * (size_t)b->num_seqs) ||
           share(r.p, n, b->page_table, 4 * (size_t)b->num_seqs * b->table_stride);
}

// What lies behind the pointers of a batch: lengths and page table, and with `rows` the rows of each sequence.  page_shift -1: no page table.
// *empty: there is nothing to do.
inline int take_seqs(const nn_kv_batch* b, int page_shift, bool rows, const char* who, KvSeqs* s, bool* empty) {
    *empty = false;
    if (b->num_seqs < 0 || (rows && b->num_rows < 0)) return NN_FAIL(NN_ERR_ARG, "%s: num_seqs=%d num_rows=%d", who, b->num_seqs, b->num_rows);
    if (b->num_seqs == 0 || (rows && b->num_rows == 0)) {
        *empty = true;
        return NN_OK;
    }
    if (b->max_len > 1 << 30) return NN_FAIL(NN_ERR_UNSUPPORTED, "%s: max_len=%d is more than 2^30", who, b->max_len);
    if ((rows && b->max_new <= 0) || b->max_len <= 0 || (page_shift >= 0 && b->table_stride <= 0))
        return NN_FAIL(NN_ERR_ARG, "%s: max_new=%d max_len=%d table_stride=%d", who, b->max_new, b->max_len, b->table_stride);
    if ((rows && !b->row_start) || !b->kv_len || (page_shift >= 0 && !b->page_table))
        return NN_FAIL(NN_ERR_ARG, "%s: null row_start, kv_len or page_table", who);
    if ((rows && !aligned(b->row_start, 4)) || !aligned(b->kv_len, 4) || (page_shift >= 0 && !aligned(b->page_table, 4)))
        return NN_FAIL(NN_ERR_ARG, "%s: row_start, kv_len and page_table must be 4-byte aligned", who);
    if (page_shift >= 0 && (long long)b->table_stride << page_shift < b->max_len)
        return NN_FAIL(NN_ERR_ARG, "%s: max_len=%d is more than a page table row of %d pages of %d positions holds", who, b->max_len, b->table_stride, 1 << page_shift);
    s->row_start = rows ? (const int*)b->row_start : nullptr;
    s->kv_len = (const int*)b->kv_len;
    s->page_table = page_shift >= 0 ? (const int*)b->page_table : nullptr;
    s->num_seqs = b->num_seqs;
    s->num_rows = rows ? b->num_rows : 0;
    s->table_stride = b->table_stride;
    s->max_len = b->max_len;
    return NN_OK;
}
inline int take_batch(nn_context* c, const nn_kv_cache* h, const nn_kv_batch* b, const char* who, KvSeqs* s, bool* empty) {
    *empty = false;
    if (!h || !b) return NN_FAIL(NN_ERR_ARG, "%s: null cache or batch", who);
    return take_seqs(b, h->view.page_shift, true, who, s, empty);
}

// Last of the checks (the others need no GPU).  The calling thread may have another device current.  h may be null: a call without a cache.
inline int make_current(nn_context* c, const nn_kv_cache* h, const char* who) {
    if (!c) return NN_FAIL(NN_ERR_ARG, "%s: null context", who);
    if (h && h->device != c->device) return NN_FAIL(NN_ERR_ARG, "%s: the cache was made for device %d, the context is of device %d", who, h->device, c->device);
    int now = -1;
    if (cudaGetDevice(&now) != cudaSuccess || now != c->device) {
        const cudaError_t e = cudaSetDevice(c->device);
        if (e != cudaSuccess) return NN_FAIL(NN_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    }
    return NN_OK;
}

// The words of a row's mask, and whether they have a bit for every new token.
inline int take_words(const nn_kv_batch* b, int words, const char* who) {
    if (words < 1 || words > TREE_MOST_WORDS) return NN_FAIL(NN_ERR_UNSUPPORTED, "%s: mask_words=%d: 1 to %d", who, words, TREE_MOST_WORDS);
    if (b->max_new > 32 * words) return NN_FAIL(NN_ERR_ARG, "%s: max_new=%d is more than the %d bits of a mask", who, b->max_new, 32 * words);
    return NN_OK;
}

}  // namespace nnb
