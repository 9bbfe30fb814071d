// Attention of new tokens over the paged key/value cache.
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

}  // namespace

cudaError_t launch_attention(const AttnArgs& a, cudaStream_t st, bool pdl) {
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
