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
// the root for one word of the mask.  Parents come before their children, so every walk ends.  26 tokens 1.4 us, 64 trees of 64 1.7, a path of 64 3.1; but each word walks for itself: a path of 256
// 61 us, one of 1024, the most that a mask has bits for, 3.5 ms (a tree of 1024 of two branches to a token 101 us).
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

// Cells go from position source[row] to the row's own, which is not behind it, as if all were read first.  A block has one head of a layer's keys or values and
// goes through the rows in order, 16 KB at a time: sources ascend, so whatever a later batch reads lies behind all that an earlier one writes, and a
// batch has been read as a whole before any of it is written.  So two batches may be on their way while the one in front of them is written: they come as
// asynchronous copies into shared memory.  Where rows are and go is found by a thread each, 256 at a time (by each of a row's 8 threads: 82 us for the case
// below, most of it instructions; with the cells in registers, which left room for two blocks of an SM, 107).
// 2048 to 1024 rows of 8 sequences, 2 heads of 64 dims of 24 layers, fp16: 58 us (5.7 TB/s), 90 with one batch after the other.  Of one sequence there are only the layers' and heads' blocks: 2048
// rows of 24 layers 17 us (the bytes 8), of one layer 12; 16000 rows 141 (60) and 82.
constexpr int MOVE_THREADS = 256, MOVE_EACH = 4, MOVE_STAGES = 3, MOVE_LISTS = 5;
struct MoveList {   // 256 rows
    int from[MOVE_THREADS], to[MOVE_THREADS];   // cell rows (a cache has less than 2^31); -1: nothing to do
    uint16_t scale[MOVE_THREADS];
};
constexpr int MOVE_BATCH = MOVE_EACH * MOVE_THREADS, MOVE_SMEM = MOVE_STAGES * MOVE_BATCH * 16 + MOVE_LISTS * (int)sizeof(MoveList);

__global__ void __launch_bounds__(MOVE_THREADS) kv_move_kernel(const __grid_constant__ KvMoveArgs a) {
    extern __shared__ __align__(16) uint8_t move_smem[];
    uint4* const held = reinterpret_cast<uint4*>(move_smem);
    MoveList* const lists = reinterpret_cast<MoveList*>(move_smem + MOVE_STAGES * MOVE_BATCH * 16);
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int cache = blockIdx.x / (2 * a.most_heads), rest = blockIdx.x - cache * 2 * a.most_heads, head = rest >> 1, tid = threadIdx.x;
    const CellRows& c = a.caches.c[cache];
    if (head >= c.kv_heads) return;
    const bool value = rest & 1;
    uint8_t* const cells = value ? c.v : c.k;
    uint16_t* const scales = value ? c.v_scale : c.k_scale;
    const int shift = a.page_shift, slots = (1 << shift) - 1, row_shift = 31 - __clz(c.row_bytes), piece_shift = row_shift - 4, per_list = piece_shift - 2;   // (1, 2 or 4 batches to a list)
    static_assert(MOVE_EACH == 4, "a batch is 1024 pieces");
    const int piece = tid & ((1 << piece_shift) - 1), my = tid >> piece_shift, rows = MOVE_THREADS >> piece_shift;   // (the same piece of every row)
    for (int s = blockIdx.y; s < a.s.num_seqs; s += gridDim.y) {
        const SeqExtent e = seq_extent(a.s.row_start[s], a.s.row_start[s + 1], a.s.kv_len[s], a.s.num_rows, a.s.max_len);
        const int n = e.row1 - e.row0, base = e.len - n;
        if (e.bad || base < 0) {
            if (tid == 0) a.status[STATUS_BAD_TABLE] = 1;
            continue;
        }
        const int* const table = a.s.page_table + (int64_t)s * a.s.table_stride;
        auto find = [&](int l) {   // list l: a row to a thread
            MoveList& list = lists[l % MOVE_LISTS];
            const int j = l * MOVE_THREADS + tid, dst = base + j;
            int from = -1, to = -1;
            if (j < n) {
                const int src = a.source[e.row0 + j], before = j > 0 ? a.source[e.row0 + j - 1] : -1;
                if (src != dst) {
                    int page = -1, to_page = -1;
                    if (src > dst && src < a.s.max_len && src > before) {
                        page = table[src >> shift];
                        to_page = table[dst >> shift];
                    }
                    if (page_ok(page, a.num_pages) && page_ok(to_page, a.num_pages)) {
                        from = (int)cell_row(page, head, src & slots, c.kv_heads, shift);
                        to = (int)cell_row(to_page, head, dst & slots, c.kv_heads, shift);
                        if (scales) list.scale[tid] = scales[from];
                    } else {
                        a.status[STATUS_BAD_TABLE] = 1;
                    }
                }
            }
            list.from[tid] = from;
            list.to[tid] = to;
        };
        const int batches = (n + MOVE_EACH * rows - 1) / (MOVE_EACH * rows);
        auto copy = [&](int b) {
            if (b < batches) {
                const MoveList& list = lists[(b >> per_list) % MOVE_LISTS];
                const uint32_t to = smem_u32(held + b % MOVE_STAGES * MOVE_BATCH + tid);
                const int r0 = (b & ((1 << per_list) - 1)) * (MOVE_EACH * rows) + my;
#pragma unroll
                for (int u = 0; u < MOVE_EACH; ++u) {
                    const int from = list.from[r0 + u * rows];
                    if (from >= 0) cp_async_16(to + u * (MOVE_THREADS * 16), cells + ((int64_t)from << row_shift) + piece * 16);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        __syncthreads();   // (the sequence before is done with the lists)
        find(0);
        find(1);
        find(2);
        find(3);
        __syncthreads();
        copy(0);
        copy(1);
        for (int b = 0; b < batches; ++b) {
            copy(b + 2);
            const bool begins = (b & ((1 << per_list) - 1)) == 0;
            asm volatile("cp.async.wait_group 2;" ::: "memory");
            __syncthreads();
            // Into the place of the list before this one's, which nobody reads behind this barrier; whoever copies its first batch does so behind the next one.
            if (begins) find((b >> per_list) + 4);
            const MoveList& list = lists[(b >> per_list) % MOVE_LISTS];
            const uint4* const mine = held + b % MOVE_STAGES * MOVE_BATCH + tid;   // (a thread writes what it has copied itself)
            const int r0 = (b & ((1 << per_list) - 1)) * (MOVE_EACH * rows) + my;
#pragma unroll
            for (int u = 0; u < MOVE_EACH; ++u) {
                const int to = list.to[r0 + u * rows];
                if (to >= 0) reinterpret_cast<uint4*>(cells + ((int64_t)to << row_shift))[piece] = mine[u * MOVE_THREADS];
            }
            if (scales && begins && list.to[tid] >= 0) scales[list.to[tid]] = list.scale[tid];
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
}

// A group's beams take over their parents' sequences.  The entries of full pages are exchanged in the table; the page that is not full will be written by each
// beam, so its cells are copied from the parent's to the beam's own.  A block takes the table, or one head of a layer's keys or values, and of it a run of
// entries or 16-byte pieces of all beams that have another parent at a time: all of them have been read before any is written, which makes any exchange
// among the beams safe without room of its own, and runs have nothing to do with one another.
// 16 groups of 8 beams of 1000 to 2000 positions (pages of 128), 2 heads of 64 dims of 24 layers, fp16: 19 us (4.3 TB/s; 21 with two pieces of a thread at a time, 23 with those of all
// beams in one thread, which left room for two blocks of an SM).
constexpr int REORDER_THREADS = 256, REORDER_EACH = 4;
// `count` values at from[m] go to to[m], for `moving` pairs of them.
template <class T>
__device__ __forceinline__ void exchange(int count, int moving, void* const* from, void* const* to) {
    const int w = 31 - __clz(REORDER_EACH * REORDER_THREADS / moving), run = 1 << w;   // places for REORDER_EACH values of each thread
    for (int i0 = 0; i0 < count; i0 += run) {
        T x[REORDER_EACH];
#pragma unroll
        for (int u = 0; u < REORDER_EACH; ++u) {
            const int place = threadIdx.x + u * REORDER_THREADS, m = place >> w, i = i0 + (place & (run - 1));
            if (m < moving && i < count) x[u] = static_cast<const T*>(from[m])[i];
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < REORDER_EACH; ++u) {
            const int place = threadIdx.x + u * REORDER_THREADS, m = place >> w, i = i0 + (place & (run - 1));
            if (m < moving && i < count) static_cast<T*>(to[m])[i] = x[u];
        }
    }
}

__global__ void __launch_bounds__(REORDER_THREADS, 6) kv_reorder_kernel(const __grid_constant__ KvReorderArgs a) {
    __shared__ void *from_at[2][MOST_BEAMS], *to_at[2][MOST_BEAMS];   // of the beams that move, one after the other: cells or table entries, and scales
    __shared__ int movers;
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int tid = threadIdx.x, lane = tid & 31, beams = a.beams, shift = a.page_shift, groups = a.s.num_seqs / beams;
    const int cache = blockIdx.x / (2 * a.most_heads), rest = blockIdx.x - cache * 2 * a.most_heads, head = rest >> 1;
    const bool tables = cache >= a.caches.n;   // this block takes the page table
    if (!tables && head >= a.caches.c[cache].kv_heads) return;
    for (int g = blockIdx.y; g < groups; g += gridDim.y) {
        __syncthreads();
        const int* const entries = a.s.page_table + (int64_t)g * beams * a.s.table_stride;
        const int len = a.s.kv_len[g * beams], full = len >> shift, rem = len & ((1 << shift) - 1);
        if (tid < 32) {
            bool good = len >= 0 && len <= a.s.max_len;
            int parent = lane, page = -1;
            if (lane < beams) {
                good = good && a.s.kv_len[g * beams + lane] == len;
                parent = a.parent[g * beams + lane];
                if (parent == -1) parent = lane;
                if (good && rem) page = entries[(int64_t)lane * a.s.table_stride + full];
                good = good && parent >= 0 && parent < beams;
            }
            good = __all_sync(0xffffffffu, good);
            const bool moves = lane < beams && parent != lane;
            const unsigned all = __ballot_sync(0xffffffffu, moves);
            const int from = __shfl_sync(0xffffffffu, page, parent & 31), at = __popc(all & ((1u << lane) - 1u));
            if (good && rem) {   // a page that is written must be there, and be no other beam's; one that is read must be there
                good = !moves || (page_ok(page, a.num_pages) && page_ok(from, a.num_pages));
                for (int b = 0; b < beams; ++b) {
                    const int other = __shfl_sync(0xffffffffu, page, b);
                    good = good && !(moves && b != lane && other == page);
                }
                good = __all_sync(0xffffffffu, good);
            }
            if (moves && good) {
                if (tables) {
                    from_at[0][at] = const_cast<int*>(entries) + (int64_t)parent * a.s.table_stride;
                    to_at[0][at] = const_cast<int*>(entries) + (int64_t)lane * a.s.table_stride;
                } else if (rem) {
                    const CellRows& c = a.caches.c[cache];
                    const int64_t from_row = cell_row(from, head, 0, c.kv_heads, shift), to_row = cell_row(page, head, 0, c.kv_heads, shift);
                    uint8_t* const cells = rest & 1 ? c.v : c.k;
                    uint16_t* const scales = rest & 1 ? c.v_scale : c.k_scale;
                    from_at[0][at] = cells + from_row * c.row_bytes;
                    to_at[0][at] = cells + to_row * c.row_bytes;
                    if (scales) {
                        from_at[1][at] = scales + from_row;
                        to_at[1][at] = scales + to_row;
                    }
                }
            }
            if (lane == 0) {
                movers = good ? __popc(all) : 0;
                if (!good) a.status[STATUS_BAD_TABLE] = 1;
            }
        }
        __syncthreads();
        if (movers == 0) continue;
        if (tables) {
            exchange<int>(full, movers, from_at[0], to_at[0]);
            continue;
        }
        const CellRows& c = a.caches.c[cache];
        exchange<uint4>(rem * (c.row_bytes / 16), movers, from_at[0], to_at[0]);
        if (c.k_scale) exchange<uint16_t>(rem, movers, from_at[1], to_at[1]);
    }
}

template <class Args>
cudaError_t launch(void (*kernel)(const Args), const Args& a, dim3 grid, int threads, int smem, cudaStream_t st, bool pdl) {
    cudaLaunchConfig_t cfg = {};
    cfg.dynamicSmemBytes = (size_t)smem;
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
    return launch(tree_layout_kernel, a, dim3((unsigned)(a.s.num_seqs < 65535 ? a.s.num_seqs : 65535)), LAYOUT_THREADS, 0, st, pdl);
}

cudaError_t branch_configure() { return cudaFuncSetAttribute(kv_move_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOVE_SMEM); }

cudaError_t launch_kv_move(const KvMoveArgs& a, cudaStream_t st, bool pdl) {
    return launch(kv_move_kernel, a, dim3((unsigned)(a.caches.n * 2 * a.most_heads), (unsigned)(a.s.num_seqs < 65535 ? a.s.num_seqs : 65535)), MOVE_THREADS, MOVE_SMEM, st, pdl);
}

cudaError_t launch_kv_reorder(const KvReorderArgs& a, cudaStream_t st, bool pdl) {
    const int groups = a.s.num_seqs / a.beams;
    const dim3 grid((unsigned)(a.caches.n * 2 * a.most_heads + (a.with_table ? 1 : 0)), (unsigned)(groups < 65535 ? groups : 65535));
    return launch(kv_reorder_kernel, a, grid, REORDER_THREADS, 0, st, pdl);
}

}  // namespace nnb
