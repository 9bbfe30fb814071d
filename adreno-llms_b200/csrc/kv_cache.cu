// The paged key/value cache: rotated and quantised rows are written (fused_rope_kvwrite_m1,
// src/models/smollm2-135m-instruct/src/layers/attention.cpp:724-769, writes one fp16 row) and read back.
//
//   y1 = half(x1 c - x2 s), y2 = half(x2 c + x1 s)      dims i and i + rotary / 2 of queries and keys, c and s of the row's position;
//                                                       products and sums are rounded to 32 bits one by one
//   scale = the smallest fp16 with scale * Q >= max|y|  over the row's dims; Q = 127 or 448, the largest code (row_scale)
//   code = rint(y / scale), or y / scale in e4m3        the division and the rounding exact, so that equal rows give equal codes
//   read back: half(code * scale)                       the product is exact in 32 bits
//
// Both are bound by the bytes they move, a short call by its chain of dependent loads (row starts, page number, cell).
#include "kv_cells.cuh"

namespace nnb {
namespace {

// A row of one head is D / 16 threads, each with two pieces of 8 values: with rotation the pieces i and i + rotary / 16, whose dims turn
// together, behind it neighbours.
__device__ __forceinline__ void piece_pair(int j, int rotary, int& a, int& b) {
    const int pairs = rotary / 16;
    a = j < pairs ? j : rotary / 8 + 2 * (j - pairs);
    b = j < pairs ? j + pairs : a + 1;
}

__device__ __forceinline__ void unpack8(const uint4& q, float (&f)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 p = half2_floats(w[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
    }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(floats_half2(f[0], f[1]), floats_half2(f[2], f[3]), floats_half2(f[4], f[5]), floats_half2(f[6], f[7]));
}

template <int FMT>
__device__ __forceinline__ uint2 encode8(const float (&f)[8], float scale) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (FMT == KV_INT8) {
            uint32_t u = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) u |= ((uint32_t)__float2int_rn(__fdiv_rn(f[4 * h + i], scale)) & 0xFFu) << (8 * i);
            w[h] = u;
        } else {
            const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(f[4 * h], scale), __fdiv_rn(f[4 * h + 1], scale)), __NV_SATFINITE, __NV_E4M3);
            const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(f[4 * h + 2], scale), __fdiv_rn(f[4 * h + 3], scale)), __NV_SATFINITE, __NV_E4M3);
            w[h] = (uint32_t)lo | ((uint32_t)hi << 16);
        }
    }
    return make_uint2(w[0], w[1]);
}

constexpr int WRITE_THREADS = 128;

// One block per row.
template <int FMT, int D>
__global__ void __launch_bounds__(WRITE_THREADS) kv_write_kernel(const KvWriteArgs a) {
    constexpr int LANES = D / 16;
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int r = blockIdx.x;
    const int seq = seq_of_row(a.s, r);
    if (seq >= a.s.num_seqs || r < a.s.row_start[0]) return;   // a row behind the last sequence
    const SeqExtent e = seq_extent(a.s.row_start[seq], a.s.row_start[seq + 1], a.s.kv_len[seq], a.s.num_rows, a.s.max_len);
    const int pos = e.len - (e.row1 - r);
    if (e.bad || pos < 0 || r < e.row0 || r >= e.row1 || (a.rotary && pos >= a.table_len)) {
        if (threadIdx.x == 0) *a.status = STATUS_BAD_TABLE;
        return;
    }
    const int page = a.s.page_table[(int64_t)seq * a.s.table_stride + (pos >> a.c.page_shift)];
    const bool cell = page_ok(page, a.c.num_pages);
    if (!cell && threadIdx.x == 0) *a.status = STATUS_BAD_TABLE;
    const int j = threadIdx.x % LANES;
    int pa, pb;
    piece_pair(j, a.rotary, pa, pb);
    const bool turns = j < a.rotary / 16;
    float c[8], s[8];
    if (turns) {
        const float4* ct = reinterpret_cast<const float4*>(a.cos + (int64_t)pos * (a.rotary / 2) + 8 * j);
        const float4* st = reinterpret_cast<const float4*>(a.sin + (int64_t)pos * (a.rotary / 2) + 8 * j);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float4 x = ct[i], y = st[i];
            c[4 * i] = x.x, c[4 * i + 1] = x.y, c[4 * i + 2] = x.z, c[4 * i + 3] = x.w;
            s[4 * i] = y.x, s[4 * i + 1] = y.y, s[4 * i + 2] = y.z, s[4 * i + 3] = y.w;
        }
    }
    const int nq = a.q ? a.q_heads : 0, heads = nq + 2 * a.c.kv_heads;
    for (int h0 = 0; h0 < heads; h0 += WRITE_THREADS / LANES) {   // (whole warps stay together for the shuffles)
        const int h = h0 + threadIdx.x / LANES;
        const bool on = h < heads, is_q = h < nq, is_k = !is_q && h < nq + a.c.kv_heads;
        const int hc = is_k ? h - nq : h - nq - a.c.kv_heads;
        const uint16_t* src = is_q ? a.q + r * a.q_stride + (int64_t)h * D : (is_k ? a.k + r * a.k_stride : a.v + r * a.v_stride) + (int64_t)hc * D;
        float x[8], y[8];
        if (on) {
            unpack8(reinterpret_cast<const uint4*>(src)[pa], x);
            unpack8(reinterpret_cast<const uint4*>(src)[pb], y);
            if (turns && (is_q || is_k)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float t1 = __fsub_rn(__fmul_rn(x[i], c[i]), __fmul_rn(y[i], s[i]));
                    const float t2 = __fadd_rn(__fmul_rn(y[i], c[i]), __fmul_rn(x[i], s[i]));
                    x[i] = __half2float(__float2half_rn(t1));
                    y[i] = __half2float(__float2half_rn(t2));
                }
            }
            if (is_q) {
                uint4* dst = reinterpret_cast<uint4*>(a.q_out + r * a.qo_stride + (int64_t)h * D);
                dst[pa] = pack8(x);
                dst[pb] = pack8(y);
            }
        }
        if (FMT == KV_FP16) {
            if (on && !is_q && cell) {
                const int64_t at = cell_row(page, hc, pos & ((1 << a.c.page_shift) - 1), a.c.kv_heads, a.c.page_shift);
                uint4* dst = reinterpret_cast<uint4*>((uint16_t*)(is_k ? a.c.k : a.c.v) + at * D);
                dst[pa] = pack8(x);
                dst[pb] = pack8(y);
            }
        } else {
            float most = 0.f;
            bool nan = false;
            if (on) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    most = fmaxf(most, fmaxf(fabsf(x[i]), fabsf(y[i])));
                    nan |= x[i] != x[i] || y[i] != y[i];
                }
            }
            if (nan) most = INFINITY;
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            if (on && !is_q && cell) {
                const int64_t at = cell_row(page, hc, pos & ((1 << a.c.page_shift) - 1), a.c.kv_heads, a.c.page_shift);
                const uint16_t sc = row_scale(most, kv_max_code(FMT));
                const float f = half_float(sc);
                uint2* dst = reinterpret_cast<uint2*>((uint8_t*)(is_k ? a.c.k : a.c.v) + at * D);
                const bool whole = sc != 0x7FFF;
                dst[pa] = whole ? encode8<FMT>(x, f) : make_uint2(0, 0);
                dst[pb] = whole ? encode8<FMT>(y, f) : make_uint2(0, 0);
                if (j == 0) (is_k ? a.c.k_scale : a.c.v_scale)[at] = sc;
            }
        }
    }
}

constexpr int READ_THREADS = 128;

// One block per row: a thread takes 16 bytes of the cache at a time.
template <int FMT, int D>
__global__ void __launch_bounds__(READ_THREADS) kv_read_kernel(const KvReadArgs a) {
    constexpr int PIECE = FMT == KV_FP16 ? 8 : 16, LANES = D / PIECE;   // values of a piece, pieces of a head's row
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int r = blockIdx.x;
    const int seq = seq_of_row(a.s, r);
    if (seq >= a.s.num_seqs || r < a.s.row_start[0]) return;
    const SeqExtent e = seq_extent(a.s.row_start[seq], a.s.row_start[seq + 1], a.s.kv_len[seq], a.s.num_rows, a.s.max_len);
    const int pos = e.len - (e.row1 - r);
    if (r < e.row0 || r >= e.row1) {
        if (threadIdx.x == 0) *a.status = STATUS_BAD_TABLE;
        return;
    }
    int page = -1;
    if (!e.bad && pos >= 0) page = a.s.page_table[(int64_t)seq * a.s.table_stride + (pos >> a.c.page_shift)];
    const bool cell = page_ok(page, a.c.num_pages);
    if (!cell && threadIdx.x == 0) *a.status = STATUS_BAD_TABLE;
    for (int i = threadIdx.x; i < 2 * a.c.kv_heads * LANES; i += READ_THREADS) {
        const int head = (i / LANES) % a.c.kv_heads, piece = i % LANES;
        const bool is_k = i / LANES < a.c.kv_heads;
        uint16_t* out = (is_k ? a.k_out + r * a.k_stride : a.v_out + r * a.v_stride) + (int64_t)head * D + piece * PIECE;
        uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;   // (a row without a cell reads as zeros)
        if (cell) {
            const int64_t at = cell_row(page, head, pos & ((1 << a.c.page_shift) - 1), a.c.kv_heads, a.c.page_shift);
            const uint4 raw = reinterpret_cast<const uint4*>((const uint8_t*)(is_k ? a.c.k : a.c.v) + at * (D * kv_cell_bytes(FMT)))[piece];
            if (FMT == KV_FP16) {
                lo = raw;
            } else {
                const float sc = half_float((is_k ? a.c.k_scale : a.c.v_scale)[at]);
                const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
                uint32_t h[8];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    codes_to_half2x2<FMT>(w[q], h[2 * q], h[2 * q + 1]);
#pragma unroll
                    for (int p = 2 * q; p < 2 * q + 2; ++p) {
                        const float2 f = half2_floats(h[p]);
                        h[p] = floats_half2(f.x * sc, f.y * sc);
                    }
                }
                lo = make_uint4(h[0], h[1], h[2], h[3]);
                hi = make_uint4(h[4], h[5], h[6], h[7]);
            }
        }
        reinterpret_cast<uint4*>(out)[0] = lo;
        if (FMT != KV_FP16) reinterpret_cast<uint4*>(out)[1] = hi;
    }
}

template <class Args>
cudaError_t launch(void (*kernel)(const Args), const Args& a, int grid, int threads, cudaStream_t st, bool pdl) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
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

cudaError_t launch_kv_write(const KvWriteArgs& a, cudaStream_t st, bool pdl) {
    auto k = a.c.fmt == KV_FP16 ? (a.c.dim == 64 ? kv_write_kernel<KV_FP16, 64> : kv_write_kernel<KV_FP16, 128>)
             : a.c.fmt == KV_INT8 ? (a.c.dim == 64 ? kv_write_kernel<KV_INT8, 64> : kv_write_kernel<KV_INT8, 128>)
                                  : (a.c.dim == 64 ? kv_write_kernel<KV_FP8, 64> : kv_write_kernel<KV_FP8, 128>);
    return launch(k, a, a.s.num_rows, WRITE_THREADS, st, pdl);
}

cudaError_t launch_kv_read(const KvReadArgs& a, cudaStream_t st, bool pdl) {
    auto k = a.c.fmt == KV_FP16 ? (a.c.dim == 64 ? kv_read_kernel<KV_FP16, 64> : kv_read_kernel<KV_FP16, 128>)
             : a.c.fmt == KV_INT8 ? (a.c.dim == 64 ? kv_read_kernel<KV_INT8, 64> : kv_read_kernel<KV_INT8, 128>)
                                  : (a.c.dim == 64 ? kv_read_kernel<KV_FP8, 64> : kv_read_kernel<KV_FP8, 128>);
    return launch(k, a, a.s.num_rows, READ_THREADS, st, pdl);
}

}  // namespace nnb
