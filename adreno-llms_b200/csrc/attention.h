// Launch interface of the paged key/value cache and of the attention over it.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_index.h"

namespace nnb {

struct KvView {   // one layer's cache
    void* k;
    void* v;
    uint16_t* k_scale;   // fp16 per cell row; null with KV_FP16
    uint16_t* v_scale;
    int fmt, num_pages, page_shift, kv_heads, dim;
};
struct KvSeqs {   // the sequences of a call, on the device
    const int* row_start;    // [num_seqs + 1]
    const int* kv_len;       // [num_seqs]
    const int* page_table;   // [num_seqs][table_stride]
    int num_seqs, num_rows, table_stride;
    int max_len;             // at most table_stride << page_shift
};

struct KvWriteArgs {
    KvView c;
    KvSeqs s;
    const uint16_t* q;       // null: no queries to rotate
    uint16_t* q_out;
    const uint16_t* k;
    const uint16_t* v;
    const float* cos;        // [table_len][rotary / 2]
    const float* sin;
    int table_len, rotary;   // rotary 0: no rotation
    int q_heads;
    int64_t q_stride, qo_stride, k_stride, v_stride;   // values from row to row
    int* status;
};
cudaError_t launch_kv_write(const KvWriteArgs& a, cudaStream_t st, bool pdl);

struct KvReadArgs {
    KvView c;
    KvSeqs s;
    uint16_t* k_out;
    uint16_t* v_out;
    int64_t k_stride, v_stride;
    int* status;
};
cudaError_t launch_kv_read(const KvReadArgs& a, cudaStream_t st, bool pdl);

struct AttnArgs {
    KvView c;
    KvSeqs s;
    const uint16_t* q;
    uint16_t* out;
    int q_heads, group;      // group: query heads to a kv head
    int64_t q_stride, o_stride;
    float scale;
    int window, sinks;       // window 0: none
    int* status;
    unsigned* counters;      // blocks of a shared item that have arrived (0 between launches)
    int4* items;             // shared items, by the block that begins them
    int join_here;           // (chunks) whether the last block to have a part of an item joins all of them
    void* parts;             // partial results of items that blocks share: the context's, for one call at a time
};
struct AttnMaps;
cudaError_t attention_configure();
cudaError_t launch_attention(const AttnArgs& a, const AttnMaps& maps, int max_new, int sm_count, cudaStream_t st, bool pdl, int* kernels);   // *kernels: launches
bool attention_countable(const AttnArgs& a, int max_new);   // whether the call's tiles of work surely stay below 2^30
constexpr int ATTN_MAX_BLOCKS = 256;
// What an item costs besides its key tiles, in units of them (tiles of 8 KB, and of 128 keys).  With / without, us: 4096 tokens of 32 heads to 8 of 64 dims,
// fp16 125 / 162; a token each of 64 sequences of up to 500 positions 30.6 / 34.9, of 64 of 8192 with 8 heads of 128 dims, e4m3, 146 / 150.
constexpr int ATTN_DECODE_EXTRA = 8, ATTN_CHUNK_EXTRA = 3;
constexpr size_t ATTN_DECODE_PART = 18 * 512, ATTN_CHUNK_PART = 256 * 128 * 4 + 256 * 8;   // two per block
// The workspace: counters, items, parts.
constexpr size_t ATTN_COUNTER_BYTES = ATTN_MAX_BLOCKS * sizeof(unsigned), ATTN_HEAD_BYTES = ATTN_COUNTER_BYTES + ATTN_MAX_BLOCKS * sizeof(int4);
inline size_t attention_workspace_bytes(int sm_count) { return ATTN_HEAD_BYTES + 2 * (size_t)(sm_count < ATTN_MAX_BLOCKS ? sm_count : ATTN_MAX_BLOCKS) * ATTN_CHUNK_PART; }

// Which of the context's status words says that the tables or lengths that a kernel of these was given are out of range (nn_sync reports an argument
// error).  Word 0 is for waits that ran out, of any kernel: neither hides the other.
constexpr int STATUS_BAD_TABLE = 1, STATUS_WORDS = 2;

}  // namespace nnb
