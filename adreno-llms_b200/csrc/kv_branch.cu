// Several continuations of a sequence in the paged cache: the layout of a drafted tree, cells that move to earlier positions, beams that take over
// their parents' sequences.
//
// All three only move bytes, and a short call is bound by its chain of dependent loads (lengths, page numbers, cells).  The caches of all layers share
// their page numbers, so that one launch serves them all (24 launches in a row cost 24 times what a launch costs).
#include "kv_cells.cuh"
#include "kv_branch.h"

namespace nnb {
namespace {

// mask[r] = the row itself and its ancestors, position[r] = its depth behind the sequence's end.  A block for each sequence; a thread walks from its row to
// the root for one word of the mask.  Parents come before their children, so every walk ends.
constexpr int LAYOUT_THREADS = 128;
__global__ void __launch_bounds__(LAYOUT_THREADS) tree_layout_kernel(const TreeLayoutArgs a) {
    __shared__ int parent[32 * TREE_MOST_WORDS];
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    for (int s = blockIdx.x; s < a.s.num_seqs; s += gridDim.x) {
        const SeqExtent e = seq_extent(a.s.row_start[s], a.s.row_start[s + 1], a.s.kv_len[s], a.s.num_rows, a.s.max_len);
        const int n = e.row1 - e.row0, base = e.len - n;
        if (e.bad || n > 32 * a.words || base < 0) {
            if (threadIdx.x == 0) a.status[STATUS_BAD_TABLE] = 1;
            continue;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += LAYOUT_THREADS) {
            int p = a.parent[e.row0 + i];
            if (p < -1 || p >= i) {   // counts as -1
                p = -1;
                a.status[STATUS_BAD_TABLE] = 1;
            }
            parent[i] = p;
        }
        __syncthreads();
        for (int x = threadIdx.x; x < n * a.words; x += LAYOUT_THREADS) {
            const int i = x / a.words, w = x - i * a.words;
            uint32_t bits = 0;
            int depth = -1;
            for (int up = i; up >= 0; up = parent[up], ++depth)
                if (up >> 5 == w) bits |= 1u << (up & 31);
            a.mask[(int64_t)(e.row0 + i) * a.words + w] = bits;
            if (w == 0) a.position[e.row0 + i] = base + depth;
        }
    }
}

// Cells go from position source[row] to the row's own, which is not behind it, as if all were read first: sources ascend, so whatever a later batch of
// rows reads lies behind all that this one writes, and within a batch every thread has read before any writes.
constexpr int MOVE_THREADS = 256, MOVE_AHEAD = 4;
__global__ void __launch_bounds__(MOVE_THREADS) kv_move_kernel(const __grid_constant__ KvMoveArgs a) {
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int cache = blockIdx.x / (2 * a.most_heads), rest = blockIdx.x - cache * 2 * a.most_heads, head = rest >> 1;
    const CellRows& c = a.caches.c[cache];
    if (head >= c.kv_heads) return;
    const bool value = rest & 1;
    uint8_t* const cells = value ? c.v : c.k;
    uint16_t* const scales = value ? c.v_scale : c.k_scale;
    const int shift = a.page_shift, slots = (1 << shift) - 1, pieces = c.row_bytes / 16, rows = MOVE_THREADS / pieces, piece = threadIdx.x % pieces;
    for (int s = blockIdx.y; s < a.s.num_seqs; s += gridDim.y) {
        const SeqExtent e = seq_extent(a.s.row_start[s], a.s.row_start[s + 1], a.s.kv_len[s], a.s.num_rows, a.s.max_len);
        const int n = e.row1 - e.row0, base = e.len - n;
        if (e.bad || base < 0) {
            if (threadIdx.x == 0) a.status[STATUS_BAD_TABLE] = 1;
            continue;
        }
        const int* const table = a.s.page_table + (int64_t)s * a.s.table_stride;
        for (int j0 = 0; j0 < n; j0 += rows * MOVE_AHEAD) {
            int64_t to[MOVE_AHEAD];
            uint4 x[MOVE_AHEAD];
            uint16_t sc[MOVE_AHEAD];
#pragma unroll
            for (int u = 0; u < MOVE_AHEAD; ++u) {
                const int j = j0 + u * rows + threadIdx.x / pieces;
                to[u] = -1;
                if (j >= n) continue;
                const int dst = base + j, src = a.source[e.row0 + j];
                if (src == dst) continue;
                if (src < dst || src >= a.s.max_len || (j > 0 && src <= a.source[e.row0 + j - 1])) {
                    a.status[STATUS_BAD_TABLE] = 1;
                    continue;
                }
                const int from_page = table[src >> shift], to_page = table[dst >> shift];
                if (!page_ok(from_page, c.num_pages) || !page_ok(to_page, c.num_pages)) {
                    a.status[STATUS_BAD_TABLE] = 1;
                    continue;
                }
                const int64_t from = cell_row(from_page, head, src & slots, c.kv_heads, shift);
                to[u] = cell_row(to_page, head, dst & slots, c.kv_heads, shift);
                x[u] = reinterpret_cast<const uint4*>(cells + from * c.row_bytes)[piece];
                if (scales && piece == 0) sc[u] = scales[from];
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < MOVE_AHEAD; ++u) {
                if (to[u] < 0) continue;
                reinterpret_cast<uint4*>(cells + to[u] * c.row_bytes)[piece] = x[u];
                if (scales && piece == 0) scales[to[u]] = sc[u];
            }
        }
    }
}

// A group's beams take over their parents' sequences.  The entries of full pages are exchanged in the table; the page that is not full will be written by
// each beam, so its cells are copied from the parent's to the beam's own.  A thread takes the same 16 bytes (or table entry) of all beams: it has read
// them all before it writes, which makes any exchange among the beams safe without room of its own.
constexpr int REORDER_THREADS = 128;
template <int BEAMS>
__global__ void __launch_bounds__(REORDER_THREADS) kv_reorder_kernel(const __grid_constant__ KvReorderArgs a) {
    __shared__ int parent_of[BEAMS], page_of[BEAMS], ok;
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int lane = threadIdx.x & 31, beams = a.beams, shift = a.page_shift, groups = a.s.num_seqs / beams;
    const int cache = blockIdx.x / (2 * a.most_heads), rest = blockIdx.x - cache * 2 * a.most_heads, head = rest >> 1;
    const bool tables = cache >= a.caches.n;   // this block takes the page table
    if (!tables && head >= a.caches.c[cache].kv_heads) return;
    for (int g = blockIdx.y; g < groups; g += gridDim.y) {
        __syncthreads();
        const int* const entries = a.s.page_table + (int64_t)g * beams * a.s.table_stride;
        const int len = a.s.kv_len[g * beams], full = len >> shift, rem = len & ((1 << shift) - 1);
        if (threadIdx.x < 32) {
            bool good = len >= 0 && len <= a.s.max_len;
            int parent = lane, page = -1;
            if (lane < beams) {
                good = good && a.s.kv_len[g * beams + lane] == len;
                parent = a.parent[g * beams + lane];
                if (parent == -1) parent = lane;
                good = good && parent >= 0 && parent < beams;
                if (good && rem) page = entries[(int64_t)lane * a.s.table_stride + full];
            }
            good = __all_sync(0xffffffffu, good);
            if (good && rem) {   // a page that is written must be there, and be no other beam's; one that is read must be there
                const bool moves = lane < beams && parent != lane;
                const int from = __shfl_sync(0xffffffffu, page, parent & 31);
                good = !moves || (page_ok(page, a.num_pages) && page_ok(from, a.num_pages));
                for (int b = 0; b < beams; ++b) {
                    const int other = __shfl_sync(0xffffffffu, page, b);
                    good = good && !(moves && b != lane && other == page);
                }
                good = __all_sync(0xffffffffu, good);
            }
            if (lane < beams) {
                parent_of[lane] = parent;
                page_of[lane] = page;
            }
            if (lane == 0) {
                ok = good;
                if (!good) a.status[STATUS_BAD_TABLE] = 1;
            }
        }
        __syncthreads();
        if (!ok) continue;
        if (tables) {
            int* const to = const_cast<int*>(entries);
            for (int i = threadIdx.x; i < full; i += REORDER_THREADS) {
                int x[BEAMS];
#pragma unroll
                for (int b = 0; b < BEAMS; ++b)
                    if (b < beams && parent_of[b] != b) x[b] = entries[(int64_t)parent_of[b] * a.s.table_stride + i];
#pragma unroll
                for (int b = 0; b < BEAMS; ++b)
                    if (b < beams && parent_of[b] != b) to[(int64_t)b * a.s.table_stride + i] = x[b];
            }
            continue;
        }
        const CellRows& c = a.caches.c[cache];
        uint8_t* const cells = rest & 1 ? c.v : c.k;
        uint16_t* const scales = rest & 1 ? c.v_scale : c.k_scale;
        auto row0 = [&](int b) { return cell_row(page_of[b], head, 0, c.kv_heads, shift); };
        for (int i = threadIdx.x; i < rem * (c.row_bytes / 16); i += REORDER_THREADS) {
            uint4 x[BEAMS];
#pragma unroll
            for (int b = 0; b < BEAMS; ++b)
                if (b < beams && parent_of[b] != b) x[b] = reinterpret_cast<const uint4*>(cells + row0(parent_of[b]) * c.row_bytes)[i];
#pragma unroll
            for (int b = 0; b < BEAMS; ++b)
                if (b < beams && parent_of[b] != b) reinterpret_cast<uint4*>(cells + row0(b) * c.row_bytes)[i] = x[b];
        }
        if (scales)
            for (int i = threadIdx.x; i < rem; i += REORDER_THREADS) {
                uint16_t x[BEAMS];
#pragma unroll
                for (int b = 0; b < BEAMS; ++b)
                    if (b < beams && parent_of[b] != b) x[b] = scales[row0(parent_of[b]) + i];
#pragma unroll
                for (int b = 0; b < BEAMS; ++b)
                    if (b < beams && parent_of[b] != b) scales[row0(b) + i] = x[b];
            }
    }
}

template <class Args>
cudaError_t launch(void (*kernel)(const Args), const Args& a, dim3 grid, int threads, cudaStream_t st, bool pdl) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace

cudaError_t launch_tree_layout(const TreeLayoutArgs& a, cudaStream_t st, bool pdl) {
    return launch(tree_layout_kernel, a, dim3((unsigned)(a.s.num_seqs < 65535 ? a.s.num_seqs : 65535)), LAYOUT_THREADS, st, pdl);
}

cudaError_t launch_kv_move(const KvMoveArgs& a, cudaStream_t st, bool pdl) {
    return launch(kv_move_kernel, a, dim3((unsigned)(a.caches.n * 2 * a.most_heads), (unsigned)(a.s.num_seqs < 65535 ? a.s.num_seqs : 65535)), MOVE_THREADS, st, pdl);
}

cudaError_t launch_kv_reorder(const KvReorderArgs& a, cudaStream_t st, bool pdl) {
    const int groups = a.s.num_seqs / a.beams;
    const dim3 grid((unsigned)(a.caches.n * 2 * a.most_heads + (a.with_table ? 1 : 0)), (unsigned)(groups < 65535 ? groups : 65535));
    return launch(a.beams <= 8 ? kv_reorder_kernel<8> : a.beams <= 16 ? kv_reorder_kernel<16> : kv_reorder_kernel<32>, a, grid, REORDER_THREADS, st, pdl);
}

}  // namespace nnb
