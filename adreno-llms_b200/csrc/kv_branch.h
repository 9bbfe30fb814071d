// Launch interface of what moves sequences about in the paged cache: drafted trees, cells that move, beams.
#pragma once
#include "attention.h"

namespace nnb {

struct TreeLayoutArgs {
    KvSeqs s;                // (without a page table)
    const int* parent;       // [num_rows], among the sequence's new rows; -1: none
    uint32_t* mask;          // [num_rows][words]
    int* position;           // [num_rows]
    int words;
    int* status;
};
cudaError_t launch_tree_layout(const TreeLayoutArgs& a, cudaStream_t st, bool pdl);

// The cell rows of one layer, as bytes.
struct CellRows {
    uint8_t* k;
    uint8_t* v;
    uint16_t* k_scale;   // null without scales
    uint16_t* v_scale;
    int kv_heads, row_bytes;
};
// Layers of one launch (kernel arguments may have 4 KB everywhere).
constexpr int MOST_LAYERS = 64;
struct CellRowsOfLayers {
    CellRows c[MOST_LAYERS];
    int n;
};

struct KvMoveArgs {
    CellRowsOfLayers caches;
    KvSeqs s;
    const int* source;       // [num_rows]: where the row's cells are now
    int page_shift, most_heads, num_pages;   // num_pages: the fewest of all layers
    int* status;
};
cudaError_t launch_kv_move(const KvMoveArgs& a, cudaStream_t st, bool pdl);
cudaError_t branch_configure();   // once for each device

constexpr int MOST_BEAMS = 32;
struct KvReorderArgs {
    CellRowsOfLayers caches;
    KvSeqs s;                // beam after beam, group after group
    const int* parent;       // [num_seqs], among the group's beams; -1: itself
    int beams, page_shift, most_heads, num_pages;   // num_pages: the fewest of all layers
    bool with_table;         // whether this launch exchanges the page table's entries
    int* status;
};
cudaError_t launch_kv_reorder(const KvReorderArgs& a, cudaStream_t st, bool pdl);

// The best continuations of groups of beams.
constexpr int MOST_PICKS = 32, MOST_BEAM_ROWS = 8192, MOST_VOCAB = 1 << 26;
struct BeamSelectArgs {
    const uint16_t* logits;  // [groups * beams][stride]
    int64_t stride;
    const float* score;      // [groups][beams]
    const int* done;         // [groups][beams], or null
    float* out_score;        // [groups][picks]
    int* out_token;
    int* out_parent;
    int* out_done;           // or null
    int groups, beams, vocab, picks, eos;
    int segs, per_seg;       // segments of a row, vectors of 8 values of a segment (set by the launch)
    unsigned* counters;      // [2 * MOST_BEAM_ROWS], 0 between launches: of rows, of groups
    void* rows;              // [MOST_BEAM_ROWS] candidates of rows
    void* parts;             // [BEAM_PARTS] results of segments
};
// The workspace, one call at a time: counters, rows, parts.
constexpr int BEAM_PARTS = 8192;
constexpr size_t BEAM_PART_BYTES = 4 * 256 + 16, BEAM_ROW_BYTES = 12 * MOST_PICKS, BEAM_COUNTER_BYTES = 2 * MOST_BEAM_ROWS * sizeof(unsigned),
                 BEAM_WORK_BYTES = BEAM_COUNTER_BYTES + MOST_BEAM_ROWS * BEAM_ROW_BYTES + BEAM_PARTS * BEAM_PART_BYTES;
void beam_segments(int rows, int vocab, int sm_count, int* segs, int* per_seg);
cudaError_t launch_beam_select(const BeamSelectArgs& a, int sm_count, cudaStream_t st, bool pdl);

}  // namespace nnb
