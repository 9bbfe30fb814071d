// Tensor maps of a cache's pages, made once with its handle.
#pragma once
#include <cuda.h>

#include "attention.h"

namespace nnb {

// Cell rows ([page][kv head][slot] as one dimension) in boxes of whole rows, or of halves of 128 bytes, swizzled.
struct AttnMaps {
    alignas(64) CUtensorMap k;
    alignas(64) CUtensorMap v;
    alignas(64) CUtensorMap k_tile;   // fp16: for the operands of the tensor cores
    alignas(64) CUtensorMap v_tile;
};
bool encode_attention_maps(const KvView& c, AttnMaps* maps);

bool small_tree(const AttnArgs& a, int max_new);
int attention_decode_keys(int fmt, int dim);   // keys of a stage: what a copy takes, if a page is that long
cudaError_t attention_decode_configure();
cudaError_t launch_attention_decode(const AttnArgs& a, const AttnMaps& maps, int max_new, int sm_count, cudaStream_t st, bool pdl);
cudaError_t attention_chunk_configure();
cudaError_t launch_attention_chunk(const AttnArgs& a, const AttnMaps& maps, int sm_count, cudaStream_t st, bool pdl, int* kernels);

}  // namespace nnb
