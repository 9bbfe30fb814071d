// C-ABI layer of several continuations of a sequence: drafted trees, cells that move, beams.  Checks of arguments, then a launch.
#include <algorithm>
#include <climits>
#include <string>
#include <vector>

#include "kv_api.h"
#include "kv_branch.h"

using namespace nnb;

extern "C" int nn_tree_layout(nn_context* c, const nn_kv_batch* b, nn_buf parent, int mask_words, nn_buf mask, nn_buf position) {
    const char* who = "nn_tree_layout";
    TreeLayoutArgs a = {};
    bool empty;
    if (!b) return NN_FAIL(NN_ERR_ARG, "%s: null batch", who);
    int rc;
    if ((rc = take_words(b, mask_words, who)) || (rc = take_seqs(b, -1, true, who, &a.s, &empty))) return rc;
    if (empty) return make_current(c, nullptr, who);
    if (!parent || !mask || !position) return NN_FAIL(NN_ERR_ARG, "%s: null parent, mask or position", who);
    if (!aligned(parent, 4) || !aligned(mask, 4) || !aligned(position, 4)) return NN_FAIL(NN_ERR_ARG, "%s: parent, mask and position must be 4-byte aligned", who);
    const size_t n = 4 * (size_t)b->num_rows, nm = n * mask_words, ns = 4 * ((size_t)b->num_seqs + 1), nl = 4 * (size_t)b->num_seqs;
    if (share(mask, nm, parent, n) || share(position, n, parent, n) || share(mask, nm, position, n) || share(mask, nm, b->row_start, ns) || share(mask, nm, b->kv_len, nl) ||
        share(position, n, b->row_start, ns) || share(position, n, b->kv_len, nl))
        return NN_FAIL(NN_ERR_ARG, "%s: mask, position, parent and the batch overlap", who);
    a.parent = (const int*)parent;
    a.mask = (uint32_t*)mask;
    a.position = (int*)position;
    a.words = mask_words;
    if ((rc = make_current(c, nullptr, who))) return rc;
    a.status = c->status_dev;
    ProfScope prof(c, [&] { return std::string("tree_layout_rows") + std::to_string(b->num_rows); });
    const cudaError_t e = launch_tree_layout(a, c->stream, c->use_pdl);
    if (e != cudaSuccess) return NN_FAIL(NN_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    c->in_flight.wrote(mask, nm);
    c->in_flight.wrote(position, n);
    c->launches++;
    return NN_OK;
}

// The caches of several layers that share their page numbers; *num_pages: the fewest of any, so that a page is good in all of them or in none.
static int take_caches(nn_kv_cache* const* caches, int n, const char* who, int* num_pages) {
    if (n < 0 || (n > 0 && !caches)) return NN_FAIL(NN_ERR_ARG, "%s: num_caches=%d caches=%p", who, n, (const void*)caches);
    struct Range {
        const char *lo, *hi;
    };
    std::vector<Range> all;
    try {
        all.reserve(4 * (size_t)n);
    } catch (...) {
        return NN_FAIL(NN_ERR_ARG, "%s: out of host memory", who);
    }
    *num_pages = INT_MAX;
    for (int i = 0; i < n; ++i) {
        if (!caches[i]) return NN_FAIL(NN_ERR_ARG, "%s: cache %d is null", who, i);
        const KvView& v = caches[i]->view;
        *num_pages = std::min(*num_pages, v.num_pages);
        if (v.page_shift != caches[0]->view.page_shift)
            return NN_FAIL(NN_ERR_ARG, "%s: cache %d has pages of %d positions, the first one of %d", who, i, 1 << v.page_shift, 1 << caches[0]->view.page_shift);
        if (caches[i]->device != caches[0]->device) return NN_FAIL(NN_ERR_ARG, "%s: cache %d is of another device than the first one", who, i);
        const char *k = (const char*)v.k, *w = (const char*)v.v, *ks = (const char*)v.k_scale, *vs = (const char*)v.v_scale;
        const size_t nc = cache_bytes(v), ns = scale_bytes(v);
        all.push_back(Range{k, k + nc});
        all.push_back(Range{w, w + nc});
        if (ks) all.push_back(Range{ks, ks + ns});
        if (vs) all.push_back(Range{vs, vs + ns});
    }
    const auto before = [](const Range& x, const Range& y) { return x.lo < y.lo; };
    if (!std::is_sorted(all.begin(), all.end(), before)) std::sort(all.begin(), all.end(), before);   // (30 caches: 0.6 us)
    for (size_t i = 1; i < all.size(); ++i)
        if (all[i].lo < all[i - 1].hi) return NN_FAIL(NN_ERR_ARG, "%s: two of the caches overlap", who);
    return NN_OK;
}
static CellRows cell_rows(const KvView& v) {
    return CellRows{(uint8_t*)v.k, (uint8_t*)v.v, v.k_scale, v.v_scale, v.kv_heads, v.dim * kv_cell_bytes(v.fmt)};
}
// MOST_LAYERS caches from `first` on, and the most heads of them.
static void layers_from(nn_kv_cache* const* caches, int num, int first, CellRowsOfLayers* to, int* most_heads) {
    to->n = std::min(num - first, MOST_LAYERS);
    *most_heads = 1;
    for (int i = 0; i < to->n; ++i) {
        to->c[i] = cell_rows(caches[first + i]->view);
        *most_heads = std::max(*most_heads, to->c[i].kv_heads);
    }
}
static void wrote_caches(nn_context* c, nn_kv_cache* const* caches, int n) {
    for (int i = 0; i < n; ++i) {
        const KvView& v = caches[i]->view;
        const size_t nc = cache_bytes(v), ns = scale_bytes(v);
        c->in_flight.wrote(v.k, nc);
        c->in_flight.wrote(v.v, nc);
        c->in_flight.wrote(v.k_scale, ns);
        c->in_flight.wrote(v.v_scale, ns);
    }
}

extern "C" int nn_kv_move(nn_context* c, nn_kv_cache* const* caches, int num_caches, const nn_kv_batch* b, nn_buf source) {
    const char* who = "nn_kv_move";
    KvMoveArgs a = {};
    bool empty;
    int rc = take_caches(caches, num_caches, who, &a.num_pages);
    if (rc) return rc;
    if (!b) return NN_FAIL(NN_ERR_ARG, "%s: null batch", who);
    if (num_caches == 0) return make_current(c, nullptr, who);
    a.page_shift = caches[0]->view.page_shift;
    if ((rc = take_seqs(b, a.page_shift, true, who, &a.s, &empty))) return rc;
    if (empty) return make_current(c, caches[0], who);
    if (!source || !aligned(source, 4)) return NN_FAIL(NN_ERR_ARG, "%s: source must be there and 4-byte aligned", who);
    for (int i = 0; i < num_caches; ++i)
        if (cache_over_batch(caches[i]->view, b) || over_cache(source, 4 * (size_t)b->num_rows, caches[i]->view))
            return NN_FAIL(NN_ERR_ARG, "%s: cache %d overlaps source or the batch's row_start, kv_len or page_table", who, i);
    a.source = (const int*)source;
    if ((rc = make_current(c, caches[0], who))) return rc;
    a.status = c->status_dev;
    ProfScope prof(c, [&] { return std::string("kv_move_layers") + std::to_string(num_caches) + "_rows" + std::to_string(b->num_rows); });
    for (int first = 0; first < num_caches; first += MOST_LAYERS) {
        layers_from(caches, num_caches, first, &a.caches, &a.most_heads);
        const cudaError_t e = launch_kv_move(a, c->stream, c->use_pdl);
        if (e != cudaSuccess) return NN_FAIL(NN_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
        c->launches++;
    }
    wrote_caches(c, caches, num_caches);
    return NN_OK;
}

extern "C" int nn_kv_reorder(nn_context* c, nn_kv_cache* const* caches, int num_caches, const nn_kv_batch* b, int beams, nn_buf parent) {
    const char* who = "nn_kv_reorder";
    KvReorderArgs a = {};
    bool empty;
    int rc = take_caches(caches, num_caches, who, &a.num_pages);
    if (rc) return rc;
    if (!b) return NN_FAIL(NN_ERR_ARG, "%s: null batch", who);
    if (num_caches == 0) return NN_FAIL(NN_ERR_ARG, "%s: no caches", who);
    if (beams < 1 || beams > MOST_BEAMS) return NN_FAIL(NN_ERR_UNSUPPORTED, "%s: beams=%d: 1 to %d", who, beams, MOST_BEAMS);
    a.page_shift = caches[0]->view.page_shift;
    if ((rc = take_seqs(b, a.page_shift, false, who, &a.s, &empty))) return rc;
    if (b->num_seqs % beams != 0) return NN_FAIL(NN_ERR_ARG, "%s: num_seqs=%d is not a multiple of %d beams", who, b->num_seqs, beams);
    if (empty) return make_current(c, caches[0], who);
    if (!parent || !aligned(parent, 4)) return NN_FAIL(NN_ERR_ARG, "%s: parent must be there and 4-byte aligned", who);
    const size_t n = 4 * (size_t)b->num_seqs, nt = n * b->table_stride;
    if (share(b->page_table, nt, b->kv_len, n) || share(b->page_table, nt, parent, n)) return NN_FAIL(NN_ERR_ARG, "%s: the page table, which is written, overlaps kv_len or parent", who);
    for (int i = 0; i < num_caches; ++i) {
        const KvView& v = caches[i]->view;
        if (over_cache(b->kv_len, n, v) || over_cache(b->page_table, nt, v) || over_cache(parent, n, v))
            return NN_FAIL(NN_ERR_ARG, "%s: cache %d overlaps parent, kv_len or the page table", who, i);
    }
    a.parent = (const int*)parent;
    a.beams = beams;
    if ((rc = make_current(c, caches[0], who))) return rc;
    a.status = c->status_dev;
    ProfScope prof(c, [&] { return std::string("kv_reorder_layers") + std::to_string(num_caches) + "_seqs" + std::to_string(b->num_seqs); });
    for (int first = 0; first < num_caches; first += MOST_LAYERS) {
        layers_from(caches, num_caches, first, &a.caches, &a.most_heads);
        a.with_table = first == 0;
        const cudaError_t e = launch_kv_reorder(a, c->stream, c->use_pdl);
        if (e != cudaSuccess) return NN_FAIL(NN_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
        c->launches++;
    }
    wrote_caches(c, caches, num_caches);
    c->in_flight.wrote(b->page_table, nt);
    return NN_OK;
}

// scores and flags of a group are read before its results are written: they may be the same buffers where there are as many picks as beams
extern "C" int nn_beam_select(nn_context* c, int groups, int beams, int vocab, nn_buf logits, int64_t stride, nn_buf score, nn_buf done, int eos, int picks, nn_buf out_score,
                              nn_buf out_token, nn_buf out_parent, nn_buf out_done) {
    const char* who = "nn_beam_select";
    if (groups < 0 || vocab < 1) return NN_FAIL(NN_ERR_ARG, "%s: groups=%d vocab=%d", who, groups, vocab);
    if (beams < 1 || beams > MOST_BEAMS || picks < 1 || picks > MOST_PICKS)
        return NN_FAIL(NN_ERR_UNSUPPORTED, "%s: beams=%d picks=%d: 1 to %d and 1 to %d", who, beams, picks, MOST_BEAMS, MOST_PICKS);
    if (vocab > MOST_VOCAB) return NN_FAIL(NN_ERR_UNSUPPORTED, "%s: vocab=%d is more than %d", who, vocab, MOST_VOCAB);
    if ((long long)groups * beams > MOST_BEAM_ROWS) return NN_FAIL(NN_ERR_UNSUPPORTED, "%s: %d groups of %d beams are more than %d rows", who, groups, beams, MOST_BEAM_ROWS);
    if (groups == 0) return make_current(c, nullptr, who);
    if (!logits || !score || !out_score || !out_token || !out_parent) return NN_FAIL(NN_ERR_ARG, "%s: null logits, score, out_score, out_token or out_parent", who);
    if (!aligned(logits, 2) || !aligned(score, 4) || !aligned(done, 4) || !aligned(out_score, 4) || !aligned(out_token, 4) || !aligned(out_parent, 4) || !aligned(out_done, 4))
        return NN_FAIL(NN_ERR_ARG, "%s: a buffer is not aligned to its values", who);
    if (stride == 0) stride = vocab;
    if (stride < vocab) return NN_FAIL(NN_ERR_ARG, "%s: logits_stride=%lld is less than vocab=%d", who, (long long)stride, vocab);
    if ((done || out_done) && (eos < 0 || eos >= vocab)) return NN_FAIL(NN_ERR_ARG, "%s: eos=%d with beams that end: a token below %d", who, eos, vocab);
    const size_t rows = (size_t)groups * beams, nl = ((rows - 1) * (size_t)stride + vocab) * 2, ni = 4 * rows, no = 4 * (size_t)groups * picks;
    const void* outs[4] = {out_score, out_token, out_parent, out_done};
    for (int i = 0; i < 4; ++i) {
        for (int j = 0; j < i; ++j)
            if (share(outs[i], no, outs[j], no)) return NN_FAIL(NN_ERR_ARG, "%s: two of the outputs overlap", who);
        const bool in_place_score = i == 0 && out_score == score && picks == beams, in_place_done = i == 3 && out_done == done && picks == beams;
        if (share(outs[i], no, logits, nl) || (!in_place_score && share(outs[i], no, score, ni)) || (!in_place_done && share(outs[i], no, done, ni)))
            return NN_FAIL(NN_ERR_ARG, "%s: an output overlaps logits, score or done", who);
    }
    BeamSelectArgs a = {};
    beam_segments((int)rows, vocab, c ? c->sm_count : 1, &a.segs, &a.per_seg);
    if ((long long)rows * a.segs > BEAM_PARTS)
        return NN_FAIL(NN_ERR_UNSUPPORTED, "%s: %d rows of %d logits are more than %d segments of 524288", who, (int)rows, vocab, BEAM_PARTS);
    int rc;
    if ((rc = make_current(c, nullptr, who))) return rc;
    a.counters = (unsigned*)c->beam_work;
    a.rows = (char*)c->beam_work + BEAM_COUNTER_BYTES;
    a.parts = (char*)a.rows + MOST_BEAM_ROWS * BEAM_ROW_BYTES;
    a.logits = (const uint16_t*)logits;
    a.stride = stride;
    a.score = (const float*)score;
    a.done = (const int*)done;
    a.out_score = (float*)out_score;
    a.out_token = (int*)out_token;
    a.out_parent = (int*)out_parent;
    a.out_done = (int*)out_done;
    a.groups = groups;
    a.beams = beams;
    a.vocab = vocab;
    a.picks = picks;
    a.eos = eos;
    ProfScope prof(c, [&] { return std::string("beam_select_groups") + std::to_string(groups) + "x" + std::to_string(beams) + "_n" + std::to_string(vocab); });
    const cudaError_t e = launch_beam_select(a, c->sm_count, c->stream, c->use_pdl);
    if (e != cudaSuccess) return NN_FAIL(NN_ERR_CUDA, "%s: launch failed: %s", who, cudaGetErrorString(e));
    for (const void* o : outs) c->in_flight.wrote(o, no);
    c->launches++;
    return NN_OK;
}
