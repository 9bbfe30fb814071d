// C-ABI layer of the paged key/value cache and of the attention over it: checks of arguments, then one launch.
#include <cuda_runtime.h>

#include <cmath>
#include <new>
#include <string>

#include "../../include/nnopt_b200.h"
#include "attention.h"
#include "attention_maps.h"
#include "internal.h"
#include "kernels.h"

using namespace nnb;

struct nn_kv_cache {
    int device;
    KvView view;
    AttnMaps maps;
};

static bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

static size_t cache_bytes(const KvView& v) {
    return ((size_t)v.num_pages * v.kv_heads << v.page_shift) * (size_t)v.dim * kv_cell_bytes(v.fmt);
}

#define CUDA_TRY(call)                                                                        \
    do {                                                                                      \
        cudaError_t e_ = (call);                                                              \
        if (e_ != cudaSuccess) return NN_FAIL(NN_ERR_CUDA, "%s: %s", #call, cudaGetErrorString(e_)); \
    } while (0)

// The partial results of items that several blocks share: one buffer for all calls of the context, which run one after the other.
// Made with the context's first cache, or by its first nn_attention on the cache of another context; the context's device is current.
static int attention_workspace(nn_context* c, const char* who) {
    if (c->attn_work) return NN_OK;
    if (c->capturing)
        return NN_FAIL(NN_ERR_UNSUPPORTED, "%s: the attention's workspace cannot be made while a plan is being recorded (the context's first cache, or its first nn_attention, makes it)", who);
    CUDA_TRY(attention_configure());
    void* work = nullptr;
    CUDA_TRY(cudaMalloc(&work, attention_workspace_bytes(c->sm_count)));
    const cudaError_t e = cudaMemsetAsync(work, 0, ATTN_HEAD_BYTES, c->stream);
    if (e != cudaSuccess) {
        cudaFree(work);
        return NN_FAIL(NN_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    }
    c->attn_work = work;
    return NN_OK;
}

// Rows of `width` values at a distance of `stride`.
struct Rows {
    const uint16_t* p;
    int64_t stride, width;
};
static size_t rows_bytes(const Rows& r, int rows) { return ((size_t)(rows - 1) * r.stride + r.width) * 2; }

// Whether two sets of rows share memory.  Of equal stride they may be columns of one buffer (q, k and v of a fused projection).
static bool rows_overlap(const Rows& a, const Rows& b, int rows) {
    const char *pa = (const char*)a.p, *pb = (const char*)b.p;
    if (pa >= pb + rows_bytes(b, rows) || pb >= pa + rows_bytes(a, rows)) return false;
    if (a.stride != b.stride) return true;
    const int64_t pitch = a.stride * 2;
    int64_t d = (int64_t)((intptr_t)pb - (intptr_t)pa) % pitch;
    if (d < 0) d += pitch;
    return d < a.width * 2 || d + b.width * 2 > pitch;
}
static bool share(const void* p, size_t np, const void* q, size_t nq) { return p && q && (const char*)p < (const char*)q + nq && (const char*)q < (const char*)p + np; }
static size_t scale_bytes(const KvView& v) { return cache_bytes(v) / ((size_t)v.dim * kv_cell_bytes(v.fmt)) * 2; }
static bool over_cache(const void* p, size_t n, const KvView& v) {
    const size_t nc = cache_bytes(v), ns = scale_bytes(v);
    return share(p, n, v.k, nc) || share(p, n, v.v, nc) || share(p, n, v.k_scale, ns) || share(p, n, v.v_scale, ns);
}
static bool rows_over_cache(const Rows& r, int rows, const KvView& v) { return over_cache(r.p, rows_bytes(r, rows), v); }
// (what a call writes must not be what tells it where to)
static bool cache_over_batch(const KvView& v, const nn_kv_batch* b) {
    return over_cache(b->row_start, 4 * ((size_t)b->num_seqs + 1), v) || over_cache(b->kv_len, 4 * (size_t)b->num_seqs, v) ||
           over_cache(b->page_table, 4 * (size_t)b->num_seqs * b->table_stride, v);
}
static bool rows_over_batch(const Rows& r, const nn_kv_batch* b) {
    const size_t n = rows_bytes(r, b->num_rows);
    return share(r.p, n, b->row_start, 4 * ((size_t)b->num_seqs + 1)) || share(r.p, n, b->kv_len, 4 * (size_t)b->num_seqs) ||
           share(r.p, n, b->page_table, 4 * (size_t)b->num_seqs * b->table_stride);
}

extern "C" int nn_kv_cache_create(nn_context* c, int format, int num_pages, int page_size, int kv_heads, int head_dim, nn_buf k, nn_buf v,
                                  nn_buf k_scale, nn_buf v_scale, nn_kv_cache** out) {
    if (!out) return NN_FAIL(NN_ERR_ARG, "nn_kv_cache_create: out is null");
    *out = nullptr;
    if (format != NN_KV_FP16 && format != NN_KV_INT8 && format != NN_KV_FP8) return NN_FAIL(NN_ERR_ARG, "nn_kv_cache_create: unknown format %d", format);
    if (num_pages <= 0 || kv_heads <= 0) return NN_FAIL(NN_ERR_ARG, "nn_kv_cache_create: bad shape num_pages=%d kv_heads=%d", num_pages, kv_heads);
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
        return NN_FAIL(NN_ERR_UNSUPPORTED, "nn_kv_cache_create: page_size=%d is none of 16, 32, 64, 128, 256", page_size);
    if (head_dim != 64 && head_dim != 128) return NN_FAIL(NN_ERR_UNSUPPORTED, "nn_kv_cache_create: head_dim=%d is neither 64 nor 128", head_dim);
    if ((long long)num_pages * page_size > 0x7FFFFFFFll / kv_heads)
        return NN_FAIL(NN_ERR_UNSUPPORTED, "nn_kv_cache_create: %d pages of %d positions and %d heads are more than 2^31 - 1 cells", num_pages, page_size, kv_heads);
    if (!k || !v) return NN_FAIL(NN_ERR_ARG, "nn_kv_cache_create: null pages (k=%p v=%p)", k, v);
    const bool scaled = format != NN_KV_FP16;
    if (scaled != (k_scale != nullptr) || scaled != (v_scale != nullptr))
        return NN_FAIL(NN_ERR_ARG, "nn_kv_cache_create: %s", scaled ? "an 8-bit cache needs both scale buffers" : "an fp16 cache has no scale buffers");
    if (!aligned(k, 16) || !aligned(v, 16) || !aligned(k_scale, 16) || !aligned(v_scale, 16))
        return NN_FAIL(NN_ERR_ARG, "nn_kv_cache_create: pages and scales must be 16-byte aligned");
    KvView w = {};
    w.k = k;
    w.v = v;
    w.k_scale = (uint16_t*)k_scale;
    w.v_scale = (uint16_t*)v_scale;
    w.fmt = format == NN_KV_FP16 ? KV_FP16 : format == NN_KV_INT8 ? KV_INT8 : KV_FP8;
    w.num_pages = num_pages;
    for (w.page_shift = 0; (1 << w.page_shift) < page_size;) ++w.page_shift;
    w.kv_heads = kv_heads;
    w.dim = head_dim;
    const size_t n = cache_bytes(w), ns = scale_bytes(w);
    if (share(k, n, v, n) || share(k_scale, ns, v_scale, ns) || share(k, n, k_scale, ns) || share(k, n, v_scale, ns) || share(v, n, k_scale, ns) || share(v, n, v_scale, ns))
        return NN_FAIL(NN_ERR_ARG, "nn_kv_cache_create: the buffers overlap");
    AttnMaps maps = {};
    if (c) {
        CUDA_TRY(cudaSetDevice(c->device));
        const int rc = attention_workspace(c, "nn_kv_cache_create");
        if (rc) return rc;
        if (!encode_attention_maps(w, &maps)) return NN_FAIL(NN_ERR_CUDA, "nn_kv_cache_create: no tensor maps for these pages (k=%p v=%p)", k, v);
    }
    nn_kv_cache* h = new (std::nothrow) nn_kv_cache{c ? c->device : -1, w, maps};
    if (!h) return NN_FAIL(NN_ERR_ARG, "nn_kv_cache_create: out of host memory");
    *out = h;
    return NN_OK;
}

extern "C" int nn_kv_cache_free(nn_kv_cache* h) {
    delete h;
    return NN_OK;
}

// The rows of one operand: `stride` 0 stands for dense rows.
static int take_rows(const void* p, int64_t stride, int heads, int dim, const char* who, const char* what, Rows* out) {
    out->p = (const uint16_t*)p;
    out->width = (int64_t)heads * dim;
    out->stride = stride ? stride : out->width;
    if (!p) return NN_FAIL(NN_ERR_ARG, "%s: %s is null", who, what);
    if (!aligned(p, 16)) return NN_FAIL(NN_ERR_ARG, "%s: %s must be 16-byte aligned", who, what);
    if (out->stride < out->width || out->stride % 8 != 0)
        return NN_FAIL(NN_ERR_ARG, "%s: stride %lld of %s: at least %lld values and a multiple of 8", who, (long long)stride, what, (long long)out->width);
    return NN_OK;
}

// *empty: there is nothing to do.
static int take_batch(nn_context* c, const nn_kv_cache* h, const nn_kv_batch* b, const char* who, KvSeqs* s, bool* empty) {
    *empty = false;
    if (!h || !b) return NN_FAIL(NN_ERR_ARG, "%s: null cache or batch", who);
    if (b->num_seqs < 0 || b->num_rows < 0) return NN_FAIL(NN_ERR_ARG, "%s: num_seqs=%d num_rows=%d", who, b->num_seqs, b->num_rows);
    if (b->num_seqs == 0 || b->num_rows == 0) {
        *empty = true;
        return NN_OK;
    }
    if (b->max_len > 1 << 30) return NN_FAIL(NN_ERR_UNSUPPORTED, "%s: max_len=%d is more than 2^30", who, b->max_len);
    if (b->max_new <= 0 || b->max_len <= 0 || b->table_stride <= 0)
        return NN_FAIL(NN_ERR_ARG, "%s: max_new=%d max_len=%d table_stride=%d", who, b->max_new, b->max_len, b->table_stride);
    if (!b->row_start || !b->kv_len || !b->page_table) return NN_FAIL(NN_ERR_ARG, "%s: null row_start, kv_len or page_table", who);
    if (!aligned(b->row_start, 4) || !aligned(b->kv_len, 4) || !aligned(b->page_table, 4))
        return NN_FAIL(NN_ERR_ARG, "%s: row_start, kv_len and page_table must be 4-byte aligned", who);
    if ((long long)b->table_stride << h->view.page_shift < b->max_len)
        return NN_FAIL(NN_ERR_ARG, "%s: max_len=%d is more than a page table row of %d pages of %d positions holds", who, b->max_len, b->table_stride, 1 << h->view.page_shift);
    s->row_start = (const int*)b->row_start;
    s->kv_len = (const int*)b->kv_len;
    s->page_table = (const int*)b->page_table;
    s->num_seqs = b->num_seqs;
    s->num_rows = b->num_rows;
    s->table_stride = b->table_stride;
    s->max_len = b->max_len;
    return NN_OK;
}

// Last of the checks (the others need no GPU).  The calling thread may have another device current.
static int make_current(nn_context* c, const nn_kv_cache* h, const char* who) {
    if (!c) return NN_FAIL(NN_ERR_ARG, "%s: null context", who);
    if (h->device != c->device) return NN_FAIL(NN_ERR_ARG, "%s: the cache was made for device %d, the context is of device %d", who, h->device, c->device);
    int now = -1;
    if (cudaGetDevice(&now) != cudaSuccess || now != c->device) {
        const cudaError_t e = cudaSetDevice(c->device);
        if (e != cudaSuccess) return NN_FAIL(NN_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    }
    return NN_OK;
}

static const char* kv_name(int fmt) { return fmt == KV_FP16 ? "fp16" : fmt == KV_INT8 ? "int8" : "fp8"; }

static int kv_write(nn_context* c, nn_kv_cache* h, const nn_kv_batch* b, nn_buf cos_f32, nn_buf sin_f32, int table_len, int rotary_dim, int q_heads, nn_buf q,
                    int64_t q_stride, nn_buf q_out, int64_t q_out_stride, nn_buf k, int64_t k_stride, nn_buf v, int64_t v_stride, const char* who) {
    KvWriteArgs a = {};
    bool empty;
    int rc = take_batch(c, h, b, who, &a.s, &empty);
    if (rc) return rc;
    if (empty) return make_current(c, h, who);
    a.c = h->view;
    const int D = a.c.dim;
    Rows rk, rv, rq = {}, ro = {};
    if ((rc = take_rows(k, k_stride, a.c.kv_heads, D, who, "k", &rk)) || (rc = take_rows(v, v_stride, a.c.kv_heads, D, who, "v", &rv))) return rc;
    if (q_heads < 0 || (q_heads > 0) != (q != nullptr) || (q != nullptr) != (q_out != nullptr))
        return NN_FAIL(NN_ERR_ARG, "%s: q_heads=%d with q=%p q_out=%p", who, q_heads, q, q_out);
    if (q) {
        if ((rc = take_rows(q, q_stride, q_heads, D, who, "q", &rq)) || (rc = take_rows(q_out, q_out_stride, q_heads, D, who, "q_out", &ro))) return rc;
        if (!(rq.p == ro.p && rq.stride == ro.stride) && rows_overlap(rq, ro, b->num_rows)) return NN_FAIL(NN_ERR_ARG, "%s: q_out overlaps q without being q", who);
        if (rows_overlap(ro, rk, b->num_rows) || rows_overlap(ro, rv, b->num_rows) || rows_over_cache(ro, b->num_rows, a.c) || rows_over_batch(ro, b))
            return NN_FAIL(NN_ERR_ARG, "%s: q_out overlaps k, v, the cache or the batch", who);
    }
    if (rows_over_cache(rk, b->num_rows, a.c) || rows_over_cache(rv, b->num_rows, a.c)) return NN_FAIL(NN_ERR_ARG, "%s: k or v lies in the cache", who);
    if (cache_over_batch(a.c, b)) return NN_FAIL(NN_ERR_ARG, "%s: the cache overlaps the batch's row_start, kv_len or page_table", who);
    if (rotary_dim) {
        if (rotary_dim < 0 || rotary_dim > D || rotary_dim % 16 != 0) return NN_FAIL(NN_ERR_ARG, "%s: rotary_dim=%d: a multiple of 16, at most %d", who, rotary_dim, D);
        if (!cos_f32 || !sin_f32 || !aligned(cos_f32, 16) || !aligned(sin_f32, 16)) return NN_FAIL(NN_ERR_ARG, "%s: cos and sin must be there and 16-byte aligned", who);
        if (table_len <= 0) return NN_FAIL(NN_ERR_ARG, "%s: table_len=%d", who, table_len);
        const size_t n = rows_bytes(ro, b->num_rows), table = (size_t)table_len * (rotary_dim / 2) * 4;
        if (q && (share(ro.p, n, cos_f32, table) || share(ro.p, n, sin_f32, table))) return NN_FAIL(NN_ERR_ARG, "%s: q_out overlaps cos or sin", who);
        if (over_cache(cos_f32, table, a.c) || over_cache(sin_f32, table, a.c)) return NN_FAIL(NN_ERR_ARG, "%s: the cache overlaps cos or sin", who);
    }
    a.q = rq.p;
    a.q_out = const_cast<uint16_t*>(ro.p);
    a.k = rk.p;
    a.v = rv.p;
    a.cos = (const float*)cos_f32;
    a.sin = (const float*)sin_f32;
    a.table_len = table_len;
    a.rotary = rotary_dim;
    a.q_heads = q_heads;
    a.q_stride = rq.stride;
    a.qo_stride = ro.stride;
    a.k_stride = rk.stride;
    a.v_stride = rv.stride;
    if ((rc = make_current(c, h, who))) return rc;
    a.status = c->status_dev;
    ProfScope prof(c, [&] { return std::string("kv_write_") + kv_name(a.c.fmt) + "_rows" + std::to_string(b->num_rows) + (rotary_dim ? "_rope" : ""); });
    const cudaError_t e = launch_kv_write(a, c->stream, c->use_pdl);
    if (e != cudaSuccess) return NN_FAIL(NN_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    const size_t n = cache_bytes(a.c), ns = scale_bytes(a.c);
    if (q) c->in_flight.wrote(q_out, rows_bytes(ro, b->num_rows));
    c->in_flight.wrote(a.c.k, n);
    c->in_flight.wrote(a.c.v, n);
    c->in_flight.wrote(a.c.k_scale, ns);
    c->in_flight.wrote(a.c.v_scale, ns);
    c->launches++;
    return NN_OK;
}

extern "C" int nn_kv_write(nn_context* c, nn_kv_cache* h, const nn_kv_batch* b, nn_buf k, int64_t k_stride, nn_buf v, int64_t v_stride) {
    return kv_write(c, h, b, nullptr, nullptr, 0, 0, 0, nullptr, 0, nullptr, 0, k, k_stride, v, v_stride, "nn_kv_write");
}

extern "C" int nn_rope_kv_write(nn_context* c, nn_kv_cache* h, const nn_kv_batch* b, nn_buf cos_f32, nn_buf sin_f32, int table_len, int rotary_dim, int q_heads,
                                nn_buf q, int64_t q_stride, nn_buf q_out, int64_t q_out_stride, nn_buf k, int64_t k_stride, nn_buf v, int64_t v_stride) {
    if (rotary_dim == 0) return NN_FAIL(NN_ERR_ARG, "nn_rope_kv_write: rotary_dim is 0 (nn_kv_write does not rotate)");
    return kv_write(c, h, b, cos_f32, sin_f32, table_len, rotary_dim, q_heads, q, q_stride, q_out, q_out_stride, k, k_stride, v, v_stride, "nn_rope_kv_write");
}

extern "C" int nn_kv_read(nn_context* c, nn_kv_cache* h, const nn_kv_batch* b, nn_buf k_out, int64_t k_stride, nn_buf v_out, int64_t v_stride) {
    const char* who = "nn_kv_read";
    KvReadArgs a = {};
    bool empty;
    int rc = take_batch(c, h, b, who, &a.s, &empty);
    if (rc) return rc;
    if (empty) return make_current(c, h, who);
    a.c = h->view;
    Rows rk, rv;
    if ((rc = take_rows(k_out, k_stride, a.c.kv_heads, a.c.dim, who, "k_out", &rk)) || (rc = take_rows(v_out, v_stride, a.c.kv_heads, a.c.dim, who, "v_out", &rv))) return rc;
    if (rows_overlap(rk, rv, b->num_rows) || rows_over_cache(rk, b->num_rows, a.c) || rows_over_cache(rv, b->num_rows, a.c) || rows_over_batch(rk, b) || rows_over_batch(rv, b))
        return NN_FAIL(NN_ERR_ARG, "%s: k_out, v_out, the cache and the batch overlap", who);
    a.k_out = const_cast<uint16_t*>(rk.p);
    a.v_out = const_cast<uint16_t*>(rv.p);
    a.k_stride = rk.stride;
    a.v_stride = rv.stride;
    if ((rc = make_current(c, h, who))) return rc;
    a.status = c->status_dev;
    ProfScope prof(c, [&] { return std::string("kv_read_") + kv_name(a.c.fmt) + "_rows" + std::to_string(b->num_rows); });
    const cudaError_t e = launch_kv_read(a, c->stream, c->use_pdl);
    if (e != cudaSuccess) return NN_FAIL(NN_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    c->in_flight.wrote(k_out, rows_bytes(rk, b->num_rows));
    c->in_flight.wrote(v_out, rows_bytes(rv, b->num_rows));
    c->launches++;
    return NN_OK;
}

extern "C" int nn_attention(nn_context* c, nn_kv_cache* h, const nn_kv_batch* b, int q_heads, nn_buf q, int64_t q_stride, nn_buf out, int64_t out_stride, float scale,
                            int window, int sinks) {
    const char* who = "nn_attention";
    AttnArgs a = {};
    bool empty;
    int rc = take_batch(c, h, b, who, &a.s, &empty);
    if (rc) return rc;
    if (empty) return make_current(c, h, who);
    a.c = h->view;
    if (q_heads <= 0 || q_heads % a.c.kv_heads != 0) return NN_FAIL(NN_ERR_ARG, "%s: q_heads=%d is not a multiple of the cache's %d heads", who, q_heads, a.c.kv_heads);
    Rows rq, ro;
    if ((rc = take_rows(q, q_stride, q_heads, a.c.dim, who, "q", &rq)) || (rc = take_rows(out, out_stride, q_heads, a.c.dim, who, "out", &ro))) return rc;
    if (rows_overlap(rq, ro, b->num_rows) || rows_over_cache(ro, b->num_rows, a.c) || rows_over_batch(ro, b))
        return NN_FAIL(NN_ERR_ARG, "%s: out overlaps q, the cache or the batch", who);
    if (!(scale > 0.f) || !std::isfinite(scale)) return NN_FAIL(NN_ERR_ARG, "%s: scale=%g: finite and positive", who, (double)scale);
    if (window < 0 || sinks < 0) return NN_FAIL(NN_ERR_ARG, "%s: window=%d sinks=%d", who, window, sinks);
    a.q = rq.p;
    a.out = const_cast<uint16_t*>(ro.p);
    a.q_heads = q_heads;
    a.group = q_heads / a.c.kv_heads;
    a.q_stride = rq.stride;
    a.o_stride = ro.stride;
    a.scale = scale;
    a.window = window;
    a.sinks = window ? sinks : 0;   // (without a window all keys up to the row's own are visible)
    if (!attention_countable(a, b->max_new))
        return NN_FAIL(NN_ERR_UNSUPPORTED, "%s: num_seqs=%d num_rows=%d max_len=%d: more than 2^30 tiles of work", who, b->num_seqs, b->num_rows, b->max_len);
    if ((rc = make_current(c, h, who)) || (rc = attention_workspace(c, who))) return rc;
    a.status = c->status_dev;
    ProfScope prof(c, [&] { return std::string("attention_") + kv_name(a.c.fmt) + "_seqs" + std::to_string(b->num_seqs) + "_rows" + std::to_string(b->num_rows); });
    a.counters = (unsigned*)c->attn_work;
    a.items = (int4*)((char*)c->attn_work + ATTN_COUNTER_BYTES);
    a.parts = (char*)c->attn_work + ATTN_HEAD_BYTES;
    int kernels = 0;
    const cudaError_t e = launch_attention(a, h->maps, b->max_new, c->sm_count, c->stream, c->use_pdl, &kernels);
    if (e != cudaSuccess) return NN_FAIL(NN_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    c->in_flight.wrote(out, rows_bytes(ro, b->num_rows));
    c->launches += kernels;
    return NN_OK;
}
