// Attention of one query row by one warp, straight from the formula: keys one after the other, hidden ones not read at all.
//
//   out = sum_k w_k v_k / sum_k w_k,  w_k = exp(scale q.k - m),  m the running maximum
//
// A lane holds D / 32 dims of q, of the sum and of each cell.
#pragma once
#include "kv_cells.cuh"

namespace nnb {

template <int FMT, int D>
__device__ __forceinline__ void load_cell_dims(const void* pages, const uint16_t* scales, int64_t at, int lane, float (&f)[D / 32]) {
    constexpr int N = D / 32;
    if (FMT == KV_FP16) {
        const uint32_t* p = reinterpret_cast<const uint32_t*>((const uint16_t*)pages + at * D + lane * N);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const float2 v = half2_floats(p[i]);
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    } else {
        const float sc = half_float(scales[at]);
        const uint16_t* p = reinterpret_cast<const uint16_t*>((const uint8_t*)pages + at * D + lane * N);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            uint32_t h01, h23;
            codes_to_half2x2<FMT>(p[i], h01, h23);
            const float2 v = half2_floats(h01);
            f[2 * i] = v.x * sc;
            f[2 * i + 1] = v.y * sc;
        }
    }
}

// Query head `head` of row `row`, position `pos` in sequence `seq` of length `len`; false: a page number was out of range (its keys count as hidden).
template <int FMT, int D>
__device__ bool attend_row(const AttnArgs& a, int seq, int len, int pos, int row, int head) {
    constexpr int N = D / 32;
    const int lane = threadIdx.x & 31, kv_head = head / a.group, mask = (1 << a.c.page_shift) - 1;
    const int* table = a.s.page_table + (int64_t)seq * a.s.table_stride;
    float q[N], o[N] = {}, m = -INFINITY, l = 0.f;
    bool any = false;
    load_cell_dims<KV_FP16, D>(a.q + row * a.q_stride + (int64_t)head * D, nullptr, 0, lane, q);
    const float scale = a.scale * 1.4426950408889634f;   // exponents are powers of two
    const int lo = window_begin(pos, a.window), end = min(pos + 1, len);
    bool ok = true;
    for (int key = 0; key < end; ++key) {
        if (key < lo && key >= a.sinks) key = lo;
        const int page = table[key >> a.c.page_shift];
        if (!page_ok(page, a.c.num_pages)) {
            ok = false;
            continue;
        }
        const int64_t at = cell_row(page, kv_head, key & mask, a.c.kv_heads, a.c.page_shift);
        float k[N], v[N], s = 0.f;
        load_cell_dims<FMT, D>(a.c.k, a.c.k_scale, at, lane, k);
        load_cell_dims<FMT, D>(a.c.v, a.c.v_scale, at, lane, v);
#pragma unroll
        for (int i = 0; i < N; ++i) s += q[i] * k[i];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        s *= scale;
        any = true;
        const float up = fmaxf(m, s), old = m == up ? 1.f : exp2f(m - up);
        const float w = s == -INFINITY ? 0.f : exp2f(s - up);   // (a NaN score makes w, and so the row, NaN)
        m = up;
        l = l * old + w;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = o[i] * old + w * v[i];
    }
    const float inv = any ? 1.f / l : 0.f;   // no visible key: zeros (only scores of -infinity: 0 / 0 as in the formula)
    uint32_t* out = reinterpret_cast<uint32_t*>(a.out + row * a.o_stride + (int64_t)head * D + lane * N);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) out[i] = floats_half2(o[2 * i] * inv, o[2 * i + 1] * inv);
    return ok;
}

}  // namespace nnb
