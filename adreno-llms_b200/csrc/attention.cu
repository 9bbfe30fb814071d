// Attention of new tokens over the paged key/value cache.
#include <cudaTypedefs.h>

#include "attention_maps.h"

namespace nnb {
namespace {

bool encode_cells(CUtensorMap* map, const KvView& c, void* base, int box_rows) {
    static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool found = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess;
        return (PFN_cuTensorMapEncodeTiled_v12000)(found ? fn : nullptr);
    }();
    if (!encode) return false;
    const int eb = kv_cell_bytes(c.fmt), row = c.dim * eb, cols = row > 128 ? 128 / eb : c.dim;   // (boxes of 128 bytes at most)
    const cuuint64_t dims[2] = {(cuuint64_t)c.dim, ((cuuint64_t)c.num_pages * c.kv_heads) << c.page_shift}, strides[1] = {(cuuint64_t)row};
    const cuuint32_t box[2] = {(cuuint32_t)cols, (cuuint32_t)box_rows}, one[2] = {1, 1};
    return encode(map, eb == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  cols * eb == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

bool encode_attention_maps(const KvView& c, AttnMaps* m) {
    const int keys = attention_decode_keys(c.fmt, c.dim), page = 1 << c.page_shift, box = keys < page ? keys : page;
    if (!encode_cells(&m->k, c, c.k, box) || !encode_cells(&m->v, c, c.v, box)) return false;
    return c.fmt != KV_FP16 || (encode_cells(&m->k_tile, c, c.k, page < 128 ? page : 128) && encode_cells(&m->v_tile, c, c.v, page < 128 ? page : 128));
}

cudaError_t attention_configure() {
    const cudaError_t e = attention_decode_configure();
    return e != cudaSuccess ? e : attention_chunk_configure();
}

// Few rows to a cache head go to the kernel that reads the cache once for every 16 of them, more to the one that reads it once for 256 but starts
// slower and, with codes, expands them first.  That one / this one, us, 4 cache heads:
//   rows   cells            1 x 2048        8 x 4096        32 x 8192 positions
//   16     fp16 of 64      10.6 / 14.0     14.5 / 21.6     45.5 / 66.6
//   16     fp16 of 128     16.4 / 16.1     23.2 / 26.3     88.4 / 82.8
//   16     e4m3 of 128     17.3 / 19.5     26.4 / 35.0     97.4 / 132
//   20     fp16 of 64      11.3 / 14.1     21.9 / 21.6     73.5 / 66.6
//   20     int8 of 64      14.2 / 16.2     24.8 / 27.1     86.8 / 91.3
//   20     e4m3 of 128     18.1 / 19.8     42.2 / 34.9      167 / 132
//   64     fp16 of 64      12.2 / 14.0     30.3 / 22.4      133 / 67
//   64     int8 of 64      14.9 / 16.7     34.6 / 27.8      159 / 92
static bool few_rows(const AttnArgs& a, int max_new) {
    const long long rows = (long long)a.group * max_new;
    if (a.group > 16 || rows > 64) return false;
    if (rows <= 16) return true;
    if (a.c.dim != 64) return false;
    return (double)a.s.num_seqs * a.s.max_len * a.c.kv_heads <= 65536.0 || (rows <= 32 && a.c.fmt != KV_FP16);
}

bool attention_countable(const AttnArgs& a, int max_new) {
    const bool few = few_rows(a, max_new);
    const long long tile = few ? attention_decode_keys(a.c.fmt, a.c.dim) : 128;
    const long long parts = few ? 1 : (a.group + 127) / 128, group = (a.group + parts - 1) / parts, tokens = few ? 8 / a.group > 0 ? 8 / a.group : 1 : 2 * (128 / group);
    const double items = (double)a.c.kv_heads * parts * ((double)a.s.num_rows / tokens + a.s.num_seqs);
    return items * ((double)a.s.max_len / tile + 2 + (few ? ATTN_DECODE_EXTRA : ATTN_CHUNK_EXTRA)) < (double)(1 << 30);
}

cudaError_t launch_attention(const AttnArgs& a, const AttnMaps& maps, int max_new, int sm_count, cudaStream_t st, bool pdl, int* kernels) {
    *kernels = 1;
    if (few_rows(a, max_new)) return launch_attention_decode(a, maps, max_new, sm_count, st, pdl);
    return launch_attention_chunk(a, maps, sm_count, st, pdl, kernels);
}

}  // namespace nnb
