// The paged key/value cache: rotated and quantised rows are written (fused_rope_kvwrite_m1,
// src/models/smollm2-135m-instruct/src/layers/attention.cpp:724-769, writes one fp16 row) and read back.
//
//   y1 = half(x1 c - x2 s), y2 = half(x2 c + x1 s)      dims i and i + rotary / 2 of queries and keys, c and s of the row's position;
//                                                       products and sums are rounded to 32 bits one by one
//   scale = the smallest fp16 with scale * Q >= max|y|  over the row's dims; Q = 127 or 448, the largest code (row_scale)
//   code = rint(y / scale), or y / scale in e4m3        rounded to nearest even, as of the exact quotient
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
__device__ __forceinline__ uint2 encode8(const float (&f)[8], float scale, float inverse) {
    // The quotient by the reciprocal, corrected by its remainder, which the fused multiply-add gives exactly (P. Markstein, IBM J. Res. Dev. 34,
    // 1990): off by less than 2^-23 of it, and exact where it is a number of 24 bits.  The values that lie between two codes are (at most 9
    // bits), and value and scale have 11 bits, so that a quotient is such a value or 2^-20 of it away.
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = f[i] * inverse;
        t[i] = copysignf(fmaf(fmaf(-q, scale, f[i]), inverse, q), f[i]);   // (-0 would lose its sign)
    }
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (FMT == KV_INT8) {
            uint32_t u = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) u |= ((uint32_t)__float2int_rn(t[4 * h + i]) & 0xFFu) << (8 * i);
            w[h] = u;
        } else {
            const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(t[4 * h], t[4 * h + 1]), __NV_SATFINITE, __NV_E4M3);
            const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(t[4 * h + 2], t[4 * h + 3]), __NV_SATFINITE, __NV_E4M3);
            w[h] = (uint32_t)lo | ((uint32_t)hi << 16);
        }
    }
    return make_uint2(w[0], w[1]);
}

// A warp per row, or four where the rows are few (SPREAD); blocks of four warps.
constexpr int WARPS = 4;

template <int FMT, int D, bool SPREAD>
__global__ void __launch_bounds__(WARPS * 32) kv_write_kernel(const KvWriteArgs a) {
    constexpr int LANES = D / 16, HEADS = 32 / LANES * (SPREAD ? WARPS : 1);   // threads of a head's row; heads at a time
    constexpr int AHEAD = SPREAD ? 1 : 3;                                      // loads of so many heads in flight
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = SPREAD ? blockIdx.x : blockIdx.x * WARPS + warp;
    if (r >= a.s.num_rows) return;
    const RowPlace at = place_of_row(a.s, r);
    if (at.none) return;
    if (at.bad || (a.rotary && at.pos >= a.table_len)) {
        if (lane == 0) a.status[STATUS_BAD_TABLE] = 1;
        return;
    }
    const int page = a.s.page_table[(int64_t)at.seq * a.s.table_stride + (at.pos >> a.c.page_shift)], slot = at.pos & ((1 << a.c.page_shift) - 1);
    const bool cell = page_ok(page, a.c.num_pages);
    if (!cell && lane == 0) a.status[STATUS_BAD_TABLE] = 1;
    const int j = lane % LANES;
    int pa, pb;
    piece_pair(j, a.rotary, pa, pb);
    const bool turns = j < a.rotary / 16;
    float c[8], s[8];
    if (turns) {
        const float4* ct = reinterpret_cast<const float4*>(a.cos + (int64_t)at.pos * (a.rotary / 2) + 8 * j);
        const float4* st = reinterpret_cast<const float4*>(a.sin + (int64_t)at.pos * (a.rotary / 2) + 8 * j);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float4 x = ct[i], y = st[i];
            c[4 * i] = x.x, c[4 * i + 1] = x.y, c[4 * i + 2] = x.z, c[4 * i + 3] = x.w;
            s[4 * i] = y.x, s[4 * i + 1] = y.y, s[4 * i + 2] = y.z, s[4 * i + 3] = y.w;
        }
    }
    const int nq = a.q ? a.q_heads : 0, heads = nq + 2 * a.c.kv_heads, first = (SPREAD ? threadIdx.x : lane) / LANES;
    for (int h0 = 0; h0 < heads; h0 += HEADS * AHEAD) {   // (whole warps stay together for the shuffles)
        uint4 in[AHEAD][2];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int h = h0 + u * HEADS + first;
            in[u][0] = in[u][1] = make_uint4(0, 0, 0, 0);
            if (h < heads) {
                const uint16_t* src = h < nq ? a.q + r * a.q_stride + (int64_t)h * D
                                             : h < nq + a.c.kv_heads ? a.k + r * a.k_stride + (int64_t)(h - nq) * D : a.v + r * a.v_stride + (int64_t)(h - nq - a.c.kv_heads) * D;
                in[u][0] = reinterpret_cast<const uint4*>(src)[pa];
                in[u][1] = reinterpret_cast<const uint4*>(src)[pb];
            }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int h = h0 + u * HEADS + first;
            const bool on = h < heads, is_q = h < nq, is_k = !is_q && h < nq + a.c.kv_heads;
            float x[8], y[8];
            unpack8(in[u][0], x);
            unpack8(in[u][1], y);
            if (turns && (is_q || is_k)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float t1 = __fsub_rn(__fmul_rn(x[i], c[i]), __fmul_rn(y[i], s[i]));
                    const float t2 = __fadd_rn(__fmul_rn(y[i], c[i]), __fmul_rn(x[i], s[i]));
                    x[i] = __half2float(__float2half_rn(t1));
                    y[i] = __half2float(__float2half_rn(t2));
                }
            }
            if (is_q) {   // (h < nq <= heads)
                uint4* dst = reinterpret_cast<uint4*>(a.q_out + r * a.qo_stride + (int64_t)h * D);
                dst[pa] = pack8(x);
                dst[pb] = pack8(y);
            }
            const bool store = on && !is_q && cell;
            const int64_t row = store ? cell_row(page, is_k ? h - nq : h - nq - a.c.kv_heads, slot, a.c.kv_heads, a.c.page_shift) : 0;
            if (FMT == KV_FP16) {
                if (store) {
                    uint4* dst = reinterpret_cast<uint4*>((uint16_t*)(is_k ? a.c.k : a.c.v) + row * D);
                    dst[pa] = pack8(x);
                    dst[pb] = pack8(y);
                }
            } else if (__any_sync(0xffffffffu, store)) {
                float most = 0.f;
                bool nan = false;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    most = fmaxf(most, fmaxf(fabsf(x[i]), fabsf(y[i])));
                    nan |= x[i] != x[i] || y[i] != y[i];
                }
                if (nan) most = INFINITY;
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                if (store) {
                    const uint16_t sc = row_scale(most, kv_max_code(FMT));
                    const float f = half_float(sc), inverse = __frcp_rn(f);
                    const bool whole = sc != 0x7FFF;
                    uint2* dst = reinterpret_cast<uint2*>((uint8_t*)(is_k ? a.c.k : a.c.v) + row * D);
                    dst[pa] = whole ? encode8<FMT>(x, f, inverse) : make_uint2(0, 0);
                    dst[pb] = whole ? encode8<FMT>(y, f, inverse) : make_uint2(0, 0);
                    if (j == 0) (is_k ? a.c.k_scale : a.c.v_scale)[row] = sc;
                }
            }
        }
    }
}

// A thread takes 16 bytes of the cache at a time, with four loads in flight.
template <int FMT, int D, bool SPREAD>
__global__ void __launch_bounds__(WARPS * 32) kv_read_kernel(const KvReadArgs a) {
    constexpr int PIECE = FMT == KV_FP16 ? 8 : 16, LANES = D / PIECE;   // values of a piece, pieces of a head's row
    constexpr int STEP = 32 * (SPREAD ? WARPS : 1), AHEAD = SPREAD ? 1 : 4;
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = SPREAD ? blockIdx.x : blockIdx.x * WARPS + warp;
    if (r >= a.s.num_rows) return;
    const RowPlace at = place_of_row(a.s, r);
    if (at.none) return;
    int page = -1;
    if (!at.bad) page = a.s.page_table[(int64_t)at.seq * a.s.table_stride + (at.pos >> a.c.page_shift)];
    const bool cell = page_ok(page, a.c.num_pages);
    if (!cell && lane == 0) a.status[STATUS_BAD_TABLE] = 1;
    const int slot = at.pos & ((1 << a.c.page_shift) - 1), all = 2 * a.c.kv_heads * LANES;
    for (int i0 = SPREAD ? threadIdx.x : lane; i0 < all; i0 += STEP * AHEAD) {
        uint4 raw[AHEAD];
        uint16_t scale[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int i = i0 + u * STEP, head = i / LANES % a.c.kv_heads;
            const bool is_k = i / LANES < a.c.kv_heads;
            raw[u] = make_uint4(0, 0, 0, 0);   // (a row without a cell reads as zeros)
            scale[u] = 0;
            if (cell && i < all) {
                const int64_t row = cell_row(page, head, slot, a.c.kv_heads, a.c.page_shift);
                raw[u] = reinterpret_cast<const uint4*>((const uint8_t*)(is_k ? a.c.k : a.c.v) + row * (D * kv_cell_bytes(FMT)))[i % LANES];
                if (FMT != KV_FP16) scale[u] = (is_k ? a.c.k_scale : a.c.v_scale)[row];
            }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int i = i0 + u * STEP, head = i / LANES % a.c.kv_heads;
            if (i >= all) break;
            const bool is_k = i / LANES < a.c.kv_heads;
            uint4* out = reinterpret_cast<uint4*>((is_k ? a.k_out + r * a.k_stride : a.v_out + r * a.v_stride) + (int64_t)head * D + i % LANES * PIECE);
            if (FMT == KV_FP16) {
                out[0] = raw[u];
                continue;
            }
            const float sc = half_float(scale[u]);
            const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
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
            out[0] = make_uint4(h[0], h[1], h[2], h[3]);
            out[1] = make_uint4(h[4], h[5], h[6], h[7]);
        }
    }
}

template <class Args>
cudaError_t launch(void (*kernel)(const Args), const Args& a, int grid, cudaStream_t st, bool pdl) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(WARPS * 32);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

// A row in four warps is ready sooner, a row in one has more loads in flight and fewer blocks to start.  Four warps / one, us, in a recorded chain of calls:
// writes of 32 + 2 x 8 heads of 128 dims, fp16: 1 row 2.5 / 4.3, 1200 rows 5.1 / 7.9, 2400 rows 8.4 / 8.1, 8192 rows 35.4 / 34.0; of 9 + 2 x 3 heads of 64:
// 1 row 1.9 / 2.1, 256 rows 2.4 / 2.3, 2400 rows 4.8 / 3.3.  Reads of 3 heads of 64 dims, int8: 1200 rows 2.5 / 2.8, 2400 rows
// 4.1 / 2.8; of 8 heads of 128 dims: 1 row 1.8 / 2.9, 2400 rows 4.6 / 7.1, 65536 rows of 16 heads, e4m3,
// 135 / 143; but of 8 heads of 64, e4m3, 70 / 50, of 4 heads of 128, fp16, 71 / 43.
constexpr int FEW_ROWS = 592;   // (four blocks for each SM)

template <int FMT, int D>
cudaError_t write_rows(const KvWriteArgs& a, cudaStream_t st, bool pdl) {
    const bool wide = ((a.q ? a.q_heads : 0) + 2 * a.c.kv_heads) * (D / 16) >= 2 * WARPS * 32;   // a row is work for four warps more than once
    if (a.s.num_rows <= (wide ? 4 * FEW_ROWS : FEW_ROWS)) return launch(kv_write_kernel<FMT, D, true>, a, a.s.num_rows, st, pdl);
    return launch(kv_write_kernel<FMT, D, false>, a, (a.s.num_rows - 1) / WARPS + 1, st, pdl);
}
template <int FMT, int D>
cudaError_t read_rows(const KvReadArgs& a, cudaStream_t st, bool pdl) {
    const bool wide = FMT != KV_FP16 && 2 * a.c.kv_heads * (D / 16) >= WARPS * 32;
    if (a.s.num_rows <= 2 * FEW_ROWS || wide) return launch(kv_read_kernel<FMT, D, true>, a, a.s.num_rows, st, pdl);
    return launch(kv_read_kernel<FMT, D, false>, a, (a.s.num_rows - 1) / WARPS + 1, st, pdl);
}

}  // namespace

cudaError_t launch_kv_write(const KvWriteArgs& a, cudaStream_t st, bool pdl) {
    if (a.c.fmt == KV_FP16) return a.c.dim == 64 ? write_rows<KV_FP16, 64>(a, st, pdl) : write_rows<KV_FP16, 128>(a, st, pdl);
    if (a.c.fmt == KV_INT8) return a.c.dim == 64 ? write_rows<KV_INT8, 64>(a, st, pdl) : write_rows<KV_INT8, 128>(a, st, pdl);
    return a.c.dim == 64 ? write_rows<KV_FP8, 64>(a, st, pdl) : write_rows<KV_FP8, 128>(a, st, pdl);
}

cudaError_t launch_kv_read(const KvReadArgs& a, cudaStream_t st, bool pdl) {
    if (a.c.fmt == KV_FP16) return a.c.dim == 64 ? read_rows<KV_FP16, 64>(a, st, pdl) : read_rows<KV_FP16, 128>(a, st, pdl);
    if (a.c.fmt == KV_INT8) return a.c.dim == 64 ? read_rows<KV_INT8, 64>(a, st, pdl) : read_rows<KV_INT8, 128>(a, st, pdl);
    return a.c.dim == 64 ? read_rows<KV_FP8, 64>(a, st, pdl) : read_rows<KV_FP8, 128>(a, st, pdl);
}

}  // namespace nnb
