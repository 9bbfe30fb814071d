// Attention of new tokens over the paged key/value cache.
#include <cudaTypedefs.h>

#include "attention_maps.h"
#include "attention_row.cuh"

namespace nnb {
namespace {

constexpr int ROW_WARPS = 4;

template <int FMT, int D>
__global__ void __launch_bounds__(ROW_WARPS * 32) attention_rows_kernel(const AttnArgs a) {
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int r = blockIdx.x;
    const int seq = seq_of_row(a.s, r);
    if (seq >= a.s.num_seqs || r < a.s.row_start[0]) return;
    const SeqExtent e = seq_extent(a.s.row_start[seq], a.s.row_start[seq + 1], a.s.kv_len[seq], a.s.num_rows, a.s.max_len);
    if (r < e.row0 || r >= e.row1) {   // (row starts that do not ascend)
        if (threadIdx.x == 0) *a.status = STATUS_BAD_TABLE;
        return;
    }
    const int head = blockIdx.y * ROW_WARPS + (threadIdx.x >> 5);
    if (head >= a.q_heads) return;
    const bool ok = attend_row<FMT, D>(a, seq, e.len, e.len - (e.row1 - r), r, head);
    if ((!ok || e.bad) && (threadIdx.x & 31) == 0) *a.status = STATUS_BAD_TABLE;
}

bool encode_cells(CUtensorMap* map, const KvView& c, void* base, int box_rows) {
    static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
    if (!encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || !fn || q != cudaDriverEntryPointSuccess) return false;
        encode = (PFN_cuTensorMapEncodeTiled_v12000)fn;
    }
    const int eb = kv_cell_bytes(c.fmt), row = c.dim * eb, cols = row > 128 ? 128 / eb : c.dim;
    const cuuint64_t dims[2] = {(cuuint64_t)c.dim, ((cuuint64_t)c.num_pages * c.kv_heads) << c.page_shift}, strides[1] = {(cuuint64_t)row};
    const cuuint32_t box[2] = {(cuuint32_t)cols, (cuuint32_t)box_rows}, one[2] = {1, 1};
    return encode(map, eb == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  cols * eb == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

bool encode_attention_maps(const KvView& c, AttnMaps* m) {
    const int keys = attention_decode_keys(c.fmt, c.dim), page = 1 << c.page_shift, box = keys < page ? keys : page;
    return encode_cells(&m->k, c, c.k, box) && encode_cells(&m->v, c, c.v, box);
}

cudaError_t attention_configure() { return attention_decode_configure(); }

cudaError_t launch_attention(const AttnArgs& a, const AttnMaps& maps, int max_new, int sm_count, cudaStream_t st, bool pdl) {
    if (a.group <= 16 && (long long)a.group * max_new <= 16) return launch_attention_decode(a, maps, sm_count, st, pdl);
    auto k = a.c.fmt == KV_FP16 ? (a.c.dim == 64 ? attention_rows_kernel<KV_FP16, 64> : attention_rows_kernel<KV_FP16, 128>)
             : a.c.fmt == KV_INT8 ? (a.c.dim == 64 ? attention_rows_kernel<KV_INT8, 64> : attention_rows_kernel<KV_INT8, 128>)
                                  : (a.c.dim == 64 ? attention_rows_kernel<KV_FP8, 64> : attention_rows_kernel<KV_FP8, 128>);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.s.num_rows, (unsigned)((a.q_heads + ROW_WARPS - 1) / ROW_WARPS));
    cfg.blockDim = dim3(ROW_WARPS * 32);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k, a);
}

}  // namespace nnb
