// Attention of one query row by one warp, straight from the formula.
//
//   out = sum_k w_k v_k / sum_k w_k,  w_k = exp(scale q.k - m),  m the running maximum
//
// A lane holds D / 32 dims of q, of the sum and of each cell.  Eight keys (of one page: the smallest has 16) are fetched together, since one after the
// other each key costs the latency of its page number and of its cell; hidden ones among them are fetched and not used.
#pragma once
#include "kv_cells.cuh"

namespace nnb {

// The D / 32 dims of a lane as they lie in memory, two to a word.
template <int FMT, int D>
struct CellDims {
    uint32_t w[D / 64];
    __device__ __forceinline__ void load(const void* pages, int64_t at, int lane) {
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
            w[i] = FMT == KV_FP16 ? reinterpret_cast<const uint32_t*>((const uint16_t*)pages + at * D)[lane * (D / 64) + i]
                                  : reinterpret_cast<const uint16_t*>((const uint8_t*)pages + at * D)[lane * (D / 64) + i];
    }
    __device__ __forceinline__ void floats(float (&f)[D / 32]) const {
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            uint32_t h = w[i], unused;
            if (FMT != KV_FP16) codes_to_half2x2<FMT>(w[i], h, unused);
            const float2 v = half2_floats(h);
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    }
};

// Query head `head` of row `row`, position `pos` in sequence `seq` of length `len` (TREE: `pos` is that of the sequence's first new token, and the row's mask
// tells which of them it sees); false: a page number was out of range (its keys count as hidden).
template <int FMT, int D, bool TREE>
__device__ bool attend_row(const AttnArgs& a, int seq, int len, int pos, int row, int head) {
    constexpr int N = D / 32, G = 8;
    const int lane = threadIdx.x & 31, kv_head = head / a.group, mask = (1 << a.c.page_shift) - 1;
    const int* table = a.s.page_table + (int64_t)seq * a.s.table_stride;
    float q[N], o[N] = {}, m = -INFINITY, l = 0.f;
    bool any = false, ok = true;
    CellDims<KV_FP16, D> qw;
    qw.load(a.q + row * a.q_stride + (int64_t)head * D, 0, lane);
    qw.floats(q);
    const float scale = a.scale * 1.4426950408889634f;   // exponents are powers of two
    const int lo = TREE ? 0 : window_begin(pos, a.window), end = TREE ? len : min(pos + 1, len);
    for (int key0 = 0; key0 < end && l == l; key0 += G) {   // (once the sum is a NaN the row is)
        if (!TREE && key0 + G <= lo && key0 >= a.sinks) key0 = lo / G * G;
        const int page = table[key0 >> a.c.page_shift];
        if (!page_ok(page, a.c.num_pages)) {
            ok = false;
            continue;
        }
        const int64_t at = cell_row(page, kv_head, key0 & mask, a.c.kv_heads, a.c.page_shift);
        CellDims<FMT, D> kc[G], vc[G];
        uint16_t ks[G], vs[G];
#pragma unroll
        for (int i = 0; i < G; ++i) {
            kc[i].load(a.c.k, at + i, lane);
            vc[i].load(a.c.v, at + i, lane);
            if (FMT != KV_FP16) {
                ks[i] = a.c.k_scale[at + i];
                vs[i] = a.c.v_scale[at + i];
            }
        }
        const uint32_t tree = TREE ? tree_bits(a.tree + (int64_t)row * a.tree_words, a.tree_words, key0, pos, len) : 0u;
        float s[G];
#pragma unroll
        for (int i = 0; i < G; ++i) {
            float k[N];
            kc[i].floats(k);
            s[i] = 0.f;
#pragma unroll
            for (int x = 0; x < N; ++x) s[i] += q[x] * (FMT == KV_FP16 ? k[x] : k[x] * half_float(ks[i]));
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1)
#pragma unroll
            for (int i = 0; i < G; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], d);
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const int key = key0 + i;
            if (TREE ? !(tree >> i & 1u) : key >= end || (key < lo && key >= a.sinks)) continue;
            any = true;
            const float t = s[i] * scale, up = fmaxf(m, t), old = m == up ? 1.f : exp2f(m - up);
            const float w = t == -INFINITY ? 0.f : exp2f(t - up);   // (a NaN score makes w, and so the row, NaN)
            m = up;
            l = l * old + w;
            float v[N];
            vc[i].floats(v);
#pragma unroll
            for (int x = 0; x < N; ++x) o[x] = o[x] * old + w * (FMT == KV_FP16 ? v[x] : v[x] * half_float(vs[i]));
        }
    }
    const float inv = any ? 1.f / l : 0.f;   // no visible key: zeros (only scores of -infinity: 0 / 0 as in the formula)
    uint32_t* out = reinterpret_cast<uint32_t*>(a.out + row * a.o_stride + (int64_t)head * D + lane * N);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) out[i] = floats_half2(o[2 * i] * inv, o[2 * i + 1] * inv);
    return ok;
}

}  // namespace nnb
