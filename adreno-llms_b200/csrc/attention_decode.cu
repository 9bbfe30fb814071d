// Attention of few new tokens: up to 8 or 16 query rows (new tokens times query heads to a cache head) read a cache head together.
//
//   t_k = scale log2(e) q.k,  w_k = 2^(t_k - m),  out = sum w_k v_k / sum w_k          m: 15 below the running maximum of t
//
// An 8-bit cell is code * scale.  The products take the codes as they are (exact in fp16), a key's scale joins its score, and a value's
// scale its weight: t'_k = t_k + log2(scale_v), w'_k = 2^(t'_k - m'), out = sum w'_k code_k / sum w'_k / scale_v, so that the weights
// that are rounded to fp16 for the second product are at most 2^15 and no rounding is added.
//
// The largest weight is 2^15 and not 1 because fp16 holds less than 11 bits of what is below 2^-14 and nothing of what is below 2^-25.  A value row of zeros has the scale 1 and
// may so have the largest w' without a part in the result: beside it nothing was left of rows of values around 0.01 (scale 2^-13) whose weights are 2^12 times smaller.
// (Scores from 2^27 on are 16 apart, and so may m be from their maximum: a weight of 2^16 is infinite, and such a row is computed once more.)
//
// Bound by the bytes of the cache: every cell is read once, for all rows, and a cell does 4 rows flops per byte.  So: twelve warps per block and
// one block per SM, each warp with a ring of its own of 8 KB stages that tensor copies fill (16 to 64 keys with their values),
// no synchronisation between warps along the keys; the units of all sequences and heads are dealt out evenly (attention_work.cuh).
// 64 sequences of 8192 positions, 32 heads to 8 of 128 dims, e4m3: 180 us, 6.1 TB/s (a plain copy 6.55); of 4096 to 8192 positions 143 us, 5.6 TB/s, in one
// program and 157, 5.1, in another.
//
// Next to the bytes it is bound by instructions: 8 KB have 354 clocks of the SM, 1416 instructions of its four schedulers, and e4m3 codes took 1344
// as the rows of m16n8k16 products.  So keys and dims are the products' rows and the queries their 8 columns (the few rows waste no half of a
// product, a score or a sum): S^T = K Q^T and O^T += V^T W^T, codes converted in registers on the way, the weights turned around by movmatrix.
// (tcgen05 would want the codes as fp16 in shared memory, four times their traffic there.)
//
// A short call is bound by its chain of steps: of 17 thousand clocks to 700 positions (9 us) the lengths took 1100, dealing out 2500, the first
// segment 700, page numbers 700, the copies 1500, scores and weights of one stage 4000, adding up and storing the rest.
#include "attention_maps.h"
#include "attention_row.cuh"
#include "attention_work.cuh"

namespace nnb {
namespace {

constexpr int WARPS = 12, STAGES = 2, STAGE = 8192, PART = STAGE / 2, THREADS = WARPS * 32;
// A row that is computed once more from the formula takes 130 to 200 ns a key, an item of 16 rows 350: 0.4 s at this length, of the 2 s that the next launch's
// waits have.  Where rows may be longer, that launch begins when this one has ended.
constexpr int MOST_KEYS_ONCE_MORE = 1 << 20;

template <int FMT, int D>
struct Shape {
    static constexpr int EB = kv_cell_bytes(FMT), ROW = D * EB, KT = PART / ROW;   // bytes of a cell row, keys of a stage
    static constexpr int KG = KT / 16, DG = D / 16;                                // groups of 16 keys, of 16 dims
};
constexpr int S_RING = 0, S_SCALE = WARPS * STAGES * STAGE, S_MERGE = S_SCALE + WARPS * STAGES * 256, MERGE_BYTES = 25344, S_BARS = S_MERGE + MERGE_BYTES,
              S_HERE = S_BARS + WARPS * STAGES * 8, S_FLAG = S_HERE + WARPS * STAGES * 4, SMEM_BYTES = S_FLAG + 32 + 1024;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");

__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
// 8 x 8 values of 16 bits turned around: rows lane / 4, columns 2 (lane % 4) ..
__device__ __forceinline__ uint32_t turned(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Bytes 0 and 2, and bytes 1 and 3, of four codes as half2, exact.
template <int FMT>
__device__ __forceinline__ void codes_even_odd(uint32_t w, uint32_t& even, uint32_t& odd) {
    if (FMT == KV_INT8) {   // the bytes, their sign bit turned over, as the low mantissa bits of 1024.0h, less 1152
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const uint32_t e = (w & 0x00FF00FFu) ^ 0x64806480u, o = (w >> 8 & 0x00FF00FFu) ^ 0x64806480u;
        const __half2 he = __hsub2(*reinterpret_cast<const __half2*>(&e), bias), ho = __hsub2(*reinterpret_cast<const __half2*>(&o), bias);
        even = *reinterpret_cast<const uint32_t*>(&he);
        odd = *reinterpret_cast<const uint32_t*>(&ho);
    } else {
        const uint32_t p = __byte_perm(w, 0u, 0x3120);
        even = e4m3x2_to_half2(p & 0xFFFFu);
        odd = e4m3x2_to_half2(p >> 16);
    }
}

// Address of 16 bytes of a cell row in a stage's half, as the tensor copies' swizzle leaves them: 64-byte rows, or 128-byte rows (256-byte ones as two halves).
template <int FMT, int D>
__device__ __forceinline__ uint32_t chunk_at(uint32_t base, int row, int chunk) {
    using S = Shape<FMT, D>;
    if (S::ROW == 64) return base + row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
    return base + (chunk >> 3) * (S::KT * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

// A warp's running result: for each tile b of 8 query rows, rows 8 b + 2 (lane % 4) and + 1, and of the sums two dims of each 16:
// lane / 4 and + 8 (fp16), 2 (lane / 4) and + 1 (8-bit): o[b][g] = {first dim, row 0; row 1; second dim, row 0; row 1}.
template <int D, int NB>
struct State {
    float m[NB][2], l[NB][2];
    float4 o[NB][D / 16];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            m[b][0] = m[b][1] = -INFINITY;
            l[b][0] = l[b][1] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[b][i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    // (the sums of the weights are kept per lane along the keys)
    __device__ __forceinline__ void close() {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[b][h] += __shfl_xor_sync(0xffffffffu, l[b][h], d);
    }
    // A partial result: maxima and sums of [NB][4] pairs of rows, [NB][D / 16] quads of 32 lanes.
    __device__ __forceinline__ void store(float4* p) const {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (lane < 4) p[b * 4 + lane] = make_float4(m[b][0], l[b][0], m[b][1], l[b][1]);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) p[NB * 4 + (b * (D / 16) + i) * 32 + lane] = o[b][i];
        }
    }
    __device__ __forceinline__ void rescale(int b, float f0, float f1) {
        l[b][0] *= f0;
        l[b][1] *= f1;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            o[b][i].x *= f0;
            o[b][i].y *= f1;
            o[b][i].z *= f0;
            o[b][i].w *= f1;
        }
    }
};

// A quad of a partial result with its two rows' maxima and sums.
struct Quad {
    float4 v, h;
};
__device__ __forceinline__ Quad no_quad() { return Quad{make_float4(0.f, 0.f, 0.f, 0.f), make_float4(-INFINITY, 0.f, -INFINITY, 0.f)}; }
// q and quad k of the NB * quads of this lane of `count` partial results added up, in order; `at(i)`: the i-th of them.
template <int NB, class At>
__device__ __forceinline__ Quad add_up(Quad q, int k, int quads, int count, At&& at) {
    const int lane = threadIdx.x & 31, b = k / quads;
    constexpr int N = 4;   // (so many at once: their loads and exponentials do not wait for one another)
#pragma unroll 1
    for (int i0 = 0; i0 < count; i0 += N) {
        float4 h[N], v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float4* p = at(min(i0 + i, count - 1));
            h[i] = p[b * 4 + (lane & 3)];
            v[i] = p[NB * 4 + k * 32 + lane];
        }
        float u0 = q.h.x, u1 = q.h.z;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (i0 + i >= count) h[i].x = h[i].z = -INFINITY;
            u0 = fmaxf(u0, h[i].x);
            u1 = fmaxf(u1, h[i].z);
        }
        const float r0 = u0 == -INFINITY ? 0.f : u0, r1 = u1 == -INFINITY ? 0.f : u1, a0 = ex2(q.h.x - r0), a1 = ex2(q.h.z - r1);
        q.h = make_float4(u0, q.h.y * a0, u1, q.h.w * a1);
        q.v = make_float4(q.v.x * a0, q.v.y * a1, q.v.z * a0, q.v.w * a1);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float f0 = ex2(h[i].x - r0), f1 = ex2(h[i].z - r1);
            q.h.y = fmaf(h[i].y, f0, q.h.y);
            q.h.w = fmaf(h[i].w, f1, q.h.w);
            q.v = make_float4(fmaf(v[i].x, f0, q.v.x), fmaf(v[i].y, f1, q.v.y), fmaf(v[i].z, f0, q.v.z), fmaf(v[i].w, f1, q.v.w));
        }
    }
    return q;
}

template <int FMT, int D, int NB>
__global__ void __launch_bounds__(THREADS, 1) attention_decode_kernel(const __grid_constant__ AttnMaps maps, const AttnArgs a) {
    using S = Shape<FMT, D>;
    constexpr bool CODES = FMT != KV_FP16;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t base = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), quad = lane >> 2, c = lane & 3;
    const uint32_t ring = base + S_RING + warp * (STAGES * STAGE), scales = base + S_SCALE + warp * (STAGES * 256), bars = base + S_BARS + warp * (STAGES * 8);
    if (lane < STAGES) mbar_init(bars + lane * 8, CODES ? 33 : 1);   // (the tensor copies' lane, and each lane's copy of scales)
    mbar_init_fence();
    __syncwarp();
    pdl_wait_prior_grid();

    WorkShape w;
    w.group = a.group;
    w.tokens = 8 * NB / a.group;
    w.vheads = a.c.kv_heads;
    w.tile = S::KT;
    w.window = a.window;
    w.sinks = a.sinks;
    w.extra = ATTN_DECODE_EXTRA;
    Walk walk = find_work(a.s, &w, WARPS, a.status);
    if (walk.u >= walk.end) return;

    const int shift = a.c.page_shift, box = min(S::KT, 1 << shift), nbox = S::KT / box, box_shift = 31 - __clz(box), nbox_shift = 31 - __clz(nbox);
    const float scale2 = a.scale * 1.4426950408889634f;

    // ---- this warp's copies, a ring in front of its products ----
    Segment sg;
    bool more = walk.next(a.s, w, &sg);
    Walk pw = walk;
    const int* ptable = nullptr;
    int phead = 0, pcount = 0, pfirst = 0, psink = 0, pskip = 0, plast = -1, plo = 0;   // the segment: its key tiles, its last position, its window
    int pslice = 0, issued = 0, page_base = 0, page_reg = -1;
    bool pmore = more;
    auto copy_from = [&](const Segment& s) {
        const TileRange tr = s.tiles(w);
        ptable = a.s.page_table + (int64_t)s.seq * a.s.table_stride;
        phead = s.vhead;
        pcount = s.count;
        pfirst = s.first;
        psink = tr.sink_tiles;
        pskip = tr.first - tr.sink_tiles;
        plast = s.p1(w);
        plo = window_begin(max(s.p0(w), 0), w.window);
        pslice = warp;
        page_base = -64;   // (no page numbers yet)
    };
    if (more) copy_from(sg);
    auto issue = [&]() {   // the next stage's copies, if there is one
        while (pmore && pslice >= pcount) {
            Segment s;
            pmore = pw.next(a.s, w, &s);
            if (!pmore) {
                // Not earlier: waits of the next launch have a limit, which counts from its beginning, and this kernel may run for longer than that.  What is
                // left is short, but for rows to be computed once more.
                if (a.s.max_len <= MOST_KEYS_ONCE_MORE) pdl_launch_dependents();
                return;
            }
            copy_from(s);
        }
        if (!pmore) return;
        auto key_at = [&](int slice) { return (pfirst + slice + (pfirst + slice < psink ? 0 : pskip)) * S::KT; };
        // page numbers of this warp's next boxes, one per lane: those of its stages in the segment are numbered in order
        const int j = (pslice / WARPS) << nbox_shift;
        if (j + nbox > page_base + 32) {
            page_base = j;
            const int slice = ((j + lane) >> nbox_shift) * WARPS + warp, key = key_at(slice) + ((j + lane) & (nbox - 1)) * box;
            page_reg = -1;
            if (slice < pcount && key <= plast && (key + box > plo || key < w.sinks)) {
                const int page = ptable[key >> shift];
                page_reg = page_ok(page, a.c.num_pages) ? page : -1;
                if (page_reg < 0) a.status[STATUS_BAD_TABLE] = 1;
            }
        }
        const int page = __shfl_sync(0xffffffffu, page_reg, (j - page_base + lane) & 31);
        const bool mine = lane < nbox && page >= 0;
        const int stage = issued % STAGES;
        const uint32_t bar = bars + stage * 8, dst = ring + stage * STAGE, sdst = scales + stage * 256;
        const unsigned here = __ballot_sync(0xffffffffu, mine);   // the boxes that are copied: the others' keys count as hidden
        if (lane == 0) {
            reinterpret_cast<unsigned*>(smem + S_HERE)[warp * STAGES + stage] = here;
            mbar_arrive_expect_tx(bar, (uint32_t)(__popc(here) * box * 2 * S::ROW));
        }
        __syncwarp();
        if (mine) {
            const int64_t row = cell_row(page, phead, (key_at(pslice) + lane * box) & ((1 << shift) - 1), a.c.kv_heads, shift);
            const uint64_t pol = l2_policy_evict_normal();
            constexpr int HALVES = S::ROW > 128 ? 2 : 1, W = S::ROW / HALVES;
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
                tma_load_2d(dst + h * (S::KT * W) + lane * box * W, &maps.k, h * 64, (int)row, bar, pol);
                tma_load_2d(dst + PART + h * (S::KT * W) + lane * box * W, &maps.v, h * 64, (int)row, bar, pol);
            }
        }
        if (CODES) {   // 8 scales to a lane, plain asynchronous copies (with bulk ones, 64 sequences of 8192 positions, e4m3 of 128 dims: 149 us,
            // 146 so)
            const int x = lane % (S::KT / 8) * 8, from = __shfl_sync(0xffffffffu, page, x >> box_shift);
            if (lane < S::KT / 4 && from >= 0) {
                const int64_t row = cell_row(from, phead, (key_at(pslice) + x) & ((1 << shift) - 1), a.c.kv_heads, shift);
                cp_async_16(sdst + (lane < S::KT / 8 ? 0 : 128) + x * 2, (lane < S::KT / 8 ? a.c.k_scale : a.c.v_scale) + row);
            }
            cp_async_mbar_arrive_noinc(bar);
        }
        pslice += WARPS;
        ++issued;
    };

    int used = 0;
    bool dead = false;
    for (; more; more = walk.next(a.s, w, &sg)) {
        const int p0 = sg.p0(w), p1 = sg.p1(w), lo0 = window_begin(p0 < 0 ? 0 : p0, w.window), lo1 = window_begin(p1 < 0 ? 0 : p1, w.window);
        const TileRange tr = sg.tiles(w);
        // row r of the item: its token, its row of the operands (-1: none), its head, its position
        const int thirds = (256 + w.group - 1) / w.group;
        auto token_of = [&](int r) { return r * thirds >> 8; };   // r / w.group, for r and w.group up to 16
        auto row_of = [&](int r) {
            const int t = sg.qt * w.tokens + token_of(r);
            return r < w.tokens * w.group && t < sg.n ? sg.row0 + t : -1;
        };
        auto head_of = [&](int r) { return sg.vhead * w.group + r - token_of(r) * w.group; };
        auto pos_of = [&](int r) { return sg.len - sg.n + sg.qt * w.tokens + token_of(r); };
        int pos[NB][2];   // of this lane's rows of scores
        uint32_t q[NB][S::DG][2];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int h = 0; h < 2; ++h) pos[b][h] = row_of(8 * b + 2 * c + h) >= 0 ? pos_of(8 * b + 2 * c + h) : -1;
            const int row = row_of(8 * b + quad);
            const uint32_t* src = reinterpret_cast<const uint32_t*>(a.q + (int64_t)max(row, 0) * a.q_stride + (int64_t)head_of(8 * b + quad) * D);
#pragma unroll
            for (int k = 0; k < S::DG; ++k) {   // fp16: dims 2c and 2c + 1, and 8 behind; codes: the dims 4c .. that a word of them holds
                uint2 x = make_uint2(0, 0);
                if (row >= 0) x = CODES ? *reinterpret_cast<const uint2*>(src + 8 * k + 2 * c) : make_uint2(src[8 * k + c], src[8 * k + c + 4]);
                q[b][k][0] = x.x;
                q[b][k][1] = x.y;
            }
        }
        State<D, NB> st;
        st.clear();
#pragma unroll 1
        for (int slice = warp; slice < sg.count; slice += WARPS) {
#pragma unroll 1
            while (!dead && pmore && issued < used + STAGES) issue();
            const int stage = used % STAGES;
            if (!dead && !mbar_wait_bounded_warp(bars + stage * 8, (used / STAGES) & 1)) {
                dead = true;
                *a.status = 31;
            }
            ++used;
            const uint32_t kb = ring + stage * STAGE, vb = kb + PART, sb = scales + stage * 256;
            const int k0 = p1 < 0 ? 0 : tr.tile_at(sg.first + slice) * S::KT;
            const unsigned here = reinterpret_cast<const unsigned*>(smem + S_HERE)[warp * STAGES + stage];
            // some row does not see all of the keys
            const bool edge = here != (1u << nbox) - 1u || k0 + S::KT - 1 > p0 || (k0 < lo1 && k0 + S::KT > w.sinks);
            // a key that some row sees
            auto seen_by_some = [&](int x) { return k0 + x <= p1 && (k0 + x >= lo0 || k0 + x < w.sinks) && (here >> (x >> box_shift) & 1u); };
            if (edge) {   // values that no row sees: whatever lies there, their weight is 0 and they must not be NaN
                for (int i = lane; i < S::KT * (S::ROW / 16); i += 32) {
                    const int r = i / (S::ROW / 16);
                    if (!seen_by_some(r))
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(chunk_at<FMT, D>(vb, r, i % (S::ROW / 16))), "r"(0) : "memory");
                }
                __syncwarp();
            }
            // ---- scores: rows are keys quad and quad + 8 of 16, columns the queries ----
            float s[NB][S::KG][4];
#pragma unroll
            for (int t = 0; t < S::KG; ++t) {
#pragma unroll
                for (int b = 0; b < NB; ++b) s[b][t][0] = s[b][t][1] = s[b][t][2] = s[b][t][3] = 0.f;
                const int krow = 16 * t + (lane & 15);
#pragma unroll
                for (int j = 0; j < S::ROW / 32; ++j) {   // 32 bytes of 16 keys
                    uint32_t r[4];
                    ldsm_x4(chunk_at<FMT, D>(kb, krow, 2 * j + (lane >> 4)), r[0], r[1], r[2], r[3]);
                    if (!CODES) {
#pragma unroll
                        for (int b = 0; b < NB; ++b) mma_16816(s[b][t], r[0], r[1], r[2], r[3], q[b][j][0], q[b][j][1]);
                    } else {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            uint32_t a0, a1, a2, a3;
                            codes_to_half2x2<FMT>(r[2 * x], a0, a2);
                            codes_to_half2x2<FMT>(r[2 * x + 1], a1, a3);
#pragma unroll
                            for (int b = 0; b < NB; ++b) mma_16816(s[b][t], a0, a1, a2, a3, q[b][2 * j + x][0], q[b][2 * j + x][1]);
                        }
                    }
                }
            }
            // ---- as powers of two, with the factors of this lane's keys; the maximum ----
            float inv[S::KG][2];
            float top[NB][2];
#pragma unroll
            for (int b = 0; b < NB; ++b) top[b][0] = top[b][1] = -INFINITY;
#pragma unroll
            for (int t = 0; t < S::KG; ++t) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int x = 16 * t + 8 * h + quad;
                    float fa = scale2, fb = 0.f;
                    if (CODES) {
                        uint16_t ks, vs;
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(ks) : "r"(sb + x * 2));
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(vs) : "r"(sb + 128 + x * 2));
                        // (the scale of a cell that no row sees may be anything)
                        const bool seen = !edge || seen_by_some(x);
                        const float k = half_float(ks);
                        fa = seen ? scale2 * k : 1.f;
                        fb = seen ? fmaf(k, 0.f, lg2(half_float(vs))) : 0.f;   // (an infinite scale as a NaN: the formula knows what codes of 0 make of it)
                        inv[t][h] = ex2(-fb);
                    }
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float& y = s[b][t][2 * h + i];
                            y = CODES ? fmaf(y, fa, fb) : y * fa;
                            if (edge && !(key_visible(k0 + x, pos[b][i], w.window, w.sinks) && (here >> (x >> box_shift) & 1u))) y = -INFINITY;
                            top[b][i] = fmaxf(top[b][i], y);
                        }
                }
            }
            bool grows = false;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) top[b][i] = fmaxf(top[b][i], __shfl_xor_sync(0xffffffffu, top[b][i], d));
                    top[b][i] -= 15.f;   // (rounded once, before it is compared and kept: otherwise the same maximum may seem to grow)
                    grows |= top[b][i] > st.m[b][i];
                }
            if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const float u0 = fmaxf(st.m[b][0], top[b][0]), u1 = fmaxf(st.m[b][1], top[b][1]);
                    st.rescale(b, st.m[b][0] == -INFINITY ? 0.f : ex2(st.m[b][0] - u0), st.m[b][1] == -INFINITY ? 0.f : ex2(st.m[b][1] - u1));
                    st.m[b][0] = u0;
                    st.m[b][1] = u1;
                }
            }
            // ---- weights, and their product with the values: rows are dims ----
            uint32_t p[NB][S::KG][2];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float r0 = st.m[b][0] == -INFINITY ? 0.f : st.m[b][0], r1 = st.m[b][1] == -INFINITY ? 0.f : st.m[b][1];
#pragma unroll
                for (int t = 0; t < S::KG; ++t)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float e0 = ex2(s[b][t][2 * h] - r0), e1 = ex2(s[b][t][2 * h + 1] - r1);
                        st.l[b][0] = CODES ? fmaf(e0, inv[t][h], st.l[b][0]) : st.l[b][0] + e0;
                        st.l[b][1] = CODES ? fmaf(e1, inv[t][h], st.l[b][1]) : st.l[b][1] + e1;
                        p[b][t][h] = turned(floats_half2(e0, e1));
                    }
            }
#pragma unroll
            for (int t = 0; t < S::KG; ++t) {
                // 16 keys, 32 bytes: matrices of 8 keys x 16 bytes.  fp16: a0 (dims 0-7, keys 0-7), a1 (dims 8-15), a2 and a3 keys 8-15.  Codes: two
                // pieces of 16 dims; a word holds two dims of two keys
                const int vrow = 16 * t + (lane & 7) + (CODES ? (lane & 8) : (lane >> 4) * 8), vpiece = CODES ? lane >> 4 : lane >> 3 & 1;
#pragma unroll
                for (int j = 0; j < S::ROW / 32; ++j) {
                    uint32_t r[4];
                    ldsm_x4_t(chunk_at<FMT, D>(vb, vrow, 2 * j + vpiece), r[0], r[1], r[2], r[3]);
                    if (!CODES) {
#pragma unroll
                        for (int b = 0; b < NB; ++b) mma_16816(reinterpret_cast<float(&)[4]>(st.o[b][j]), r[0], r[1], r[2], r[3], p[b][t][0], p[b][t][1]);
                    } else {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            uint32_t a0, a1, a2, a3;
                            codes_even_odd<FMT>(r[2 * x], a0, a1);
                            codes_even_odd<FMT>(r[2 * x + 1], a2, a3);
#pragma unroll
                            for (int b = 0; b < NB; ++b) mma_16816(reinterpret_cast<float(&)[4]>(st.o[b][2 * j + x]), a0, a1, a2, a3, p[b][t][0], p[b][t][1]);
                        }
                    }
                }
            }
            if (edge) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // (the zeros above, before a copy lands there)
            __syncwarp();
        }

        // ---- the block's result of this segment: the warps' added up, as many at a time as there is room for (all of them where the rings are idle),
        // a quad of it to a warp ----
        st.close();
        const bool last = walk.u >= walk.end;
        constexpr int QUADS = D / 16, ALL = NB * QUADS, PARTIAL = NB * 64 + ALL * 512, N = (ALL + WARPS - 1) / WARPS;
        constexpr int SHARE = WARPS / ALL > 0 ? WARPS / ALL : 1, ROOM = MERGE_BYTES / PARTIAL < WARPS ? MERGE_BYTES / PARTIAL : WARPS;
        static_assert(PARTIAL <= (int)ATTN_DECODE_PART && PARTIAL <= STAGES * STAGE && SHARE * PARTIAL <= MERGE_BYTES, "partial results");
        unsigned* const bad = reinterpret_cast<unsigned*>(smem + S_FLAG) + 4;   // rows that are not finite, or see nothing
        volatile int* const flag = reinterpret_cast<volatile int*>(smem + S_FLAG);
        if (tid == 0) *bad = 0u;
        const int with = min(WARPS, sg.count), room = last ? WARPS : ROOM, stride = last ? STAGES * STAGE : PARTIAL;   // (warps that have had a slice)
        uint8_t* const dumps = smem + (last ? S_RING : S_MERGE);
        Quad x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = no_quad();
#pragma unroll 1
        for (int w0 = 0; w0 < with; w0 += room) {
            if (w0) __syncthreads();
            if (warp >= w0 && warp < min(w0 + room, with)) st.store(reinterpret_cast<float4*>(dumps + (warp - w0) * stride));
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (warp + i * WARPS < ALL)
                    x[i] = add_up<NB>(x[i], warp + i * WARPS, QUADS, min(room, with - w0), [&](int y) { return reinterpret_cast<const float4*>(dumps + y * stride); });
        }
        bool whole = sg.count == sg.total;
        if (!whole) {   // one of several blocks: the last to arrive adds the parts up, in the blocks' order
            float4* const slots = reinterpret_cast<float4*>(a.parts);
            const int b0 = (int)(sg.unit0 / w.chunk), b1 = (int)((sg.unit0 + sg.total - 1) / w.chunk);
            float4* const slot = slots + (int64_t)(2 * blockIdx.x + (sg.first == 0 ? 1 : 0)) * (ATTN_DECODE_PART / 16);
            auto put = [&](float4* d, int k, const Quad& y) {
                d[NB * 4 + k * 32 + lane] = y.v;
                if (k % QUADS == 0 && lane < 4) d[k / QUADS * 4 + lane] = y.h;
            };
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (warp + i * WARPS < ALL) put(slot, warp + i * WARPS, x[i]);
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const bool done = atomicAdd(a.counters + b0, 1u) == (unsigned)(b1 - b0);
                if (done) a.counters[b0] = 0u;
                *flag = done;
            }
            __syncthreads();
            whole = *flag != 0;
            if (whole) {
                __threadfence();
                const int n = b1 - b0 + 1, per = (n + SHARE - 1) / SHARE;
                uint8_t* const mid = smem + S_MERGE;
#pragma unroll 1
                for (int y = warp; y < ALL * SHARE; y += WARPS) {
                    const int k = y % ALL, lo = y / ALL * per;
                    put(reinterpret_cast<float4*>(mid + y / ALL * PARTIAL), k, add_up<NB>(no_quad(), k, QUADS, min(per, n - lo), [&](int i) {
                            const int b = b0 + lo + i;
                            return const_cast<const float4*>(slots) + (int64_t)(2 * b + (b == b0 ? 1 : 0)) * (ATTN_DECODE_PART / 16);
                        }));
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (warp + i * WARPS < ALL)
                        x[i] = add_up<NB>(no_quad(), warp + i * WARPS, QUADS, SHARE, [&](int y) { return reinterpret_cast<const float4*>(mid + y * PARTIAL); });
            }
        }
        if (whole) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int k = warp + i * WARPS;
                if (k < ALL) {
                    float4& v = x[i].v;
                    const float f0 = 1.f / x[i].h.y, f1 = 1.f / x[i].h.w;
                    v = make_float4(v.x * f0, v.y * f1, v.z * f0, v.w * f1);
                    const bool fine0 = x[i].h.y > 0.f && x[i].h.y < INFINITY && fabsf(v.x) < HALF_END && fabsf(v.z) < HALF_END;
                    const bool fine1 = x[i].h.w > 0.f && x[i].h.w < INFINITY && fabsf(v.y) < HALF_END && fabsf(v.w) < HALF_END;
                    const int r = k / QUADS * 8 + 2 * c;
                    if (!fine0 || !fine1) atomicOr(bad, (fine0 ? 0u : 1u << r) | (fine1 ? 0u : 2u << r));
                }
            }
            __syncthreads();
            const unsigned again = *bad;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int k = warp + i * WARPS;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = k / QUADS * 8 + 2 * c + h, row = k < ALL ? row_of(r) : -1;
                    if (row < 0 || (again >> r & 1u)) continue;
                    uint16_t* out = a.out + (int64_t)row * a.o_stride + (int64_t)head_of(r) * D + k % QUADS * 16;
                    const uint32_t two = floats_half2(h ? x[i].v.y : x[i].v.x, h ? x[i].v.w : x[i].v.z);
                    if (CODES) {
                        reinterpret_cast<uint32_t*>(out)[quad] = two;
                    } else {
                        out[quad] = (uint16_t)two;
                        out[quad + 8] = (uint16_t)(two >> 16);
                    }
                }
            }
            // ... from the formula once more, which does not touch hidden cells; a warp each
            int turn = 0;
            for (unsigned left = again; left; left &= left - 1) {
                const int r = __ffs(left) - 1, row = row_of(r);
                if (row < 0 || turn++ % WARPS != warp) continue;
                if (!attend_row<FMT, D>(a, sg.seq, sg.len, pos_of(r), row, head_of(r)) && lane == 0) a.status[STATUS_BAD_TABLE] = 1;
            }
        }
        if (!last) __syncthreads();   // (the buffers are free again)
    }
    // (after a wait that ran out: what was asked for must land before the block's memory is given back)
    if (dead)
        for (int i = issued < STAGES ? 0 : issued - STAGES; i < issued; ++i) mbar_wait_bounded_warp(bars + (i % STAGES) * 8, (i / STAGES) & 1);
}

template <int FMT, int D, int NB>
cudaError_t configure() {
    return cudaFuncSetAttribute(attention_decode_kernel<FMT, D, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
}
template <int FMT, int D>
cudaError_t configure() {
    const cudaError_t e = configure<FMT, D, 1>();
    return e != cudaSuccess ? e : configure<FMT, D, 2>();
}
template <int FMT, int D>
auto kernel(bool one_tile) {
    return one_tile ? attention_decode_kernel<FMT, D, 1> : attention_decode_kernel<FMT, D, 2>;
}

}  // namespace

cudaError_t attention_decode_configure() {
    cudaError_t e;
    if ((e = configure<KV_FP16, 64>()) != cudaSuccess || (e = configure<KV_FP16, 128>()) != cudaSuccess || (e = configure<KV_INT8, 64>()) != cudaSuccess ||
        (e = configure<KV_INT8, 128>()) != cudaSuccess || (e = configure<KV_FP8, 64>()) != cudaSuccess)
        return e;
    return configure<KV_FP8, 128>();
}

int attention_decode_keys(int fmt, int dim) { return PART / (dim * kv_cell_bytes(fmt)); }

cudaError_t launch_attention_decode(const AttnArgs& a, const AttnMaps& maps, int max_new, int sm_count, cudaStream_t st, bool pdl) {
    const bool one = (long long)a.group * max_new <= 8;   // one tile of 8 rows
    auto k = a.c.fmt == KV_FP16 ? (a.c.dim == 64 ? kernel<KV_FP16, 64>(one) : kernel<KV_FP16, 128>(one))
             : a.c.fmt == KV_INT8 ? (a.c.dim == 64 ? kernel<KV_INT8, 64>(one) : kernel<KV_INT8, 128>(one))
                                  : (a.c.dim == 64 ? kernel<KV_FP8, 64>(one) : kernel<KV_FP8, 128>(one));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(sm_count < ATTN_MAX_BLOCKS ? sm_count : ATTN_MAX_BLOCKS));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM_BYTES;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k, maps, a);
}

}  // namespace nnb
