// Attention of few new tokens: at most 16 query rows (new tokens times query heads to a cache head) read a cache head together.
//
//   t_k = scale log2(e) q.k,  w_k = 2^(t_k - m),  out = sum w_k v_k / sum w_k          m: the running maximum of t
//
// An 8-bit cell is code * scale.  The products take the codes as they are (exact in fp16), a key's scale joins its score, and a value's
// scale its weight: t'_k = t_k + log2(scale_v), w'_k = 2^(t'_k - m'), out = sum w'_k code_k / sum w'_k / scale_v, so that the weights
// that are rounded to fp16 for the second product are at most 1 and no rounding is added.
//
// Bound by the bytes of the cache: every cell is read once, for all rows, and a cell does 4 rows flops per byte.  So: eight warps per block and
// one block per SM, each warp with a ring of its own of 8 KB stages that tensor copies fill (16 to 64 keys with their values),
// no synchronisation between warps along the keys; the units of all sequences and heads are dealt out evenly (attention_work.cuh).
// Both products are mma.sync: 16 rows are an eighth of a tcgen05 tile's, and a warp keeps scores, weights and sums in registers.
#include "attention_maps.h"
#include "attention_row.cuh"
#include "attention_work.cuh"

namespace nnb {
namespace {

constexpr int WARPS = 8, STAGES = 3, STAGE = 8192, PART = STAGE / 2;
constexpr int MERGE_BYTES = 17408;   // two warps' sums of 128 dims with their maxima (four of 64)

template <int FMT, int D>
struct Shape {
    static constexpr int EB = kv_cell_bytes(FMT), ROW = D * EB, KT = PART / ROW;   // bytes of a cell row, keys of a stage
    static constexpr int NT = KT / 8, DT = D / 8;                                  // 8-key and 8-dim tiles
    static constexpr int DUMP = (DT + 1) * 512;                                    // a warp's partial result
    static constexpr int DUMPS = MERGE_BYTES / DUMP;                               // that fit the merge buffer
};

constexpr int S_RING = 0, S_SCALE = WARPS * STAGES * STAGE, S_MERGE = S_SCALE + WARPS * STAGES * 256, S_BARS = S_MERGE + MERGE_BYTES,
              S_HERE = S_BARS + WARPS * STAGES * 8, S_FLAG = S_HERE + WARPS * STAGES * 4,
              SMEM_BYTES = S_FLAG + 16 + 1024;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");
static_assert(sizeof(WorkShared) <= MERGE_BYTES, "the work list lies in the merge buffer");

__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
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

// Address of 16 bytes of a cell row in a stage's half, as the tensor copies' swizzle leaves them: 64-byte rows, or 128-byte rows (256-byte ones as two halves).
template <int FMT, int D>
__device__ __forceinline__ uint32_t chunk_at(uint32_t base, int row, int chunk) {
    using S = Shape<FMT, D>;
    if (S::ROW == 64) return base + row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
    return base + (chunk >> 3) * (S::KT * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

// A warp's running result for its rows lane / 4 and lane / 4 + 8.  Of 16 dims (8-bit cells) or two tiles of 8 (fp16): the accumulator
// layout of the products, which only the last step turns into dims.
template <int D>
struct State {
    float m[2], l[2];
    float o[D / 8][4];
    __device__ __forceinline__ void clear() {
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    }
    // (the sums of the weights are kept per lane along the keys)
    __device__ __forceinline__ void close() {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        }
    }
    // A partial result is [1 + D / 8][32 lanes] float4: maxima and sums, rows lane / 4, rows lane / 4 + 8 (only with `two`).
    __device__ __forceinline__ void store(float4* p, bool two) const {
        const int lane = threadIdx.x & 31;
        p[lane] = make_float4(m[0], l[0], m[1], l[1]);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) p[(1 + i) * 32 + lane] = make_float4(o[2 * i][0], o[2 * i][1], o[2 * i + 1][0], o[2 * i + 1][1]);
        if (two)
#pragma unroll
            for (int i = 0; i < D / 16; ++i) p[(1 + D / 16 + i) * 32 + lane] = make_float4(o[2 * i][2], o[2 * i][3], o[2 * i + 1][2], o[2 * i + 1][3]);
    }
    __device__ __forceinline__ void add(const float4* p, bool two) {
        const int lane = threadIdx.x & 31;
        const float4 h = p[lane];
        float4 v[D / 16];
#pragma unroll
        for (int i = 0; i < D / 16; ++i) v[i] = p[(1 + i) * 32 + lane];
        const float hm[2] = {h.x, h.z}, hl[2] = {h.y, h.w};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (r == 1) {
                if (!two) break;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) v[i] = p[(1 + D / 16 + i) * 32 + lane];
            }
            const float up = fmaxf(m[r], hm[r]);
            const float a = m[r] == -INFINITY ? 0.f : ex2(m[r] - up), b = hm[r] == -INFINITY ? 0.f : ex2(hm[r] - up);
            m[r] = up;
            l[r] = l[r] * a + hl[r] * b;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                o[2 * i][2 * r] = o[2 * i][2 * r] * a + v[i].x * b;
                o[2 * i][2 * r + 1] = o[2 * i][2 * r + 1] * a + v[i].y * b;
                o[2 * i + 1][2 * r] = o[2 * i + 1][2 * r] * a + v[i].z * b;
                o[2 * i + 1][2 * r + 1] = o[2 * i + 1][2 * r + 1] * a + v[i].w * b;
            }
        }
    }
};

// The warps' results added up, in a fixed order, into warp 0's.
template <int FMT, int D>
__device__ __forceinline__ void merge_warps(State<D>& st, uint8_t* buf, int warp, bool two) {
    using S = Shape<FMT, D>;
#pragma unroll 1
    for (int half = WARPS / 2; half > 0; half >>= 1) {
#pragma unroll 1
        for (int s0 = 0; s0 < half; s0 += S::DUMPS) {
            const int at = warp % half - s0;
            const bool in = warp < 2 * half && at >= 0 && at < S::DUMPS;
            float4* p = reinterpret_cast<float4*>(buf + (in ? at : 0) * S::DUMP);
            if (in && warp >= half) st.store(p, two);
            __syncthreads();
            if (in && warp < half) st.add(p, two);
            __syncthreads();
        }
    }
}

template <int FMT, int D>
__global__ void __launch_bounds__(WARPS * 32, 1) attention_decode_kernel(const __grid_constant__ AttnMaps maps, const AttnArgs a) {
    using S = Shape<FMT, D>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t base = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), quad = lane >> 2, c = lane & 3;
    const uint32_t ring = base + S_RING + warp * (STAGES * STAGE), scales = base + S_SCALE + warp * (STAGES * 256), bars = base + S_BARS + warp * (STAGES * 8);
    if (lane < STAGES) mbar_init(bars + lane * 8, 1);
    mbar_init_fence();
    pdl_launch_dependents();
    pdl_wait_prior_grid();

    WorkShape w;
    w.group = a.group;
    w.tokens = 16 / a.group;
    w.vheads = a.c.kv_heads;
    w.tile = S::KT;
    w.window = a.window;
    w.sinks = a.sinks;
    const bool two = w.group * w.tokens > 8;
    long long chunk;
    Walk walk = find_work(a.s, w, reinterpret_cast<WorkShared*>(smem + S_MERGE), WARPS, &chunk, a.status);
    __syncthreads();
    if (walk.u >= walk.end) return;

    const int shift = a.c.page_shift, box = min(S::KT, 1 << shift), nbox = S::KT / box, box_shift = 31 - __clz(box), nbox_shift = 31 - __clz(nbox);
    const float scale2 = a.scale * 1.4426950408889634f;

    // ---- this warp's copies, `ahead` stages in front of its products ----
    Walk pw = walk;
    Segment ps;
    bool pmore = pw.next(a.s, w, &ps);
    int pslice = warp, issued = 0, page_base = 0, page_reg = -1;
    bool fresh = true;   // page numbers of a new segment
    auto issue = [&]() {   // the next stage's copies, if there is one
        while (pmore && pslice >= ps.count) {
            pmore = pw.next(a.s, w, &ps);
            pslice = warp;
            fresh = true;
        }
        if (!pmore) return;
        const TileRange tr = ps.tiles(w);
        const int p0 = ps.p0(w), p1 = ps.p1(w), lo = window_begin(p0 < 0 ? 0 : p0, w.window);
        // page numbers of this warp's next boxes, one per lane
        const int j = (pslice / WARPS) * nbox;   // boxes of this warp's stages in the segment are numbered in order
        if (fresh || j + nbox > page_base + 32) {
            page_base = j;
            const int slice = ps.first + ((j + lane) >> nbox_shift) * WARPS + warp;
            page_reg = -1;
            if (slice < ps.first + ps.count && p1 >= 0) {
                const int key = tr.tile_at(slice) * S::KT + ((j + lane) & (nbox - 1)) * box;
                if (key <= p1 && (key + box > lo || key < w.sinks)) {
                    const int page = a.s.page_table[(int64_t)ps.seq * a.s.table_stride + (key >> shift)];
                    page_reg = page_ok(page, a.c.num_pages) ? page : -2;
                    if (page_reg == -2) *a.status = STATUS_BAD_TABLE;
                }
            }
            fresh = false;
        }
        const int page = __shfl_sync(0xffffffffu, page_reg, (j - page_base + lane) & 31);
        const bool mine = lane < nbox && page >= 0;
        const int stage = issued % STAGES;
        const uint32_t bar = bars + stage * 8, dst = ring + stage * STAGE, sdst = scales + stage * 256;
        const unsigned here = __ballot_sync(0xffffffffu, mine);   // the boxes that are copied: the others' keys count as hidden
        const int boxes = __popc(here);
        if (lane == 0) reinterpret_cast<unsigned*>(smem + S_HERE)[warp * STAGES + stage] = here;
        if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(boxes * box * (2 * S::ROW + (FMT == KV_FP16 ? 0 : 4))));
        __syncwarp();
        if (mine) {
            const int slot = (p1 < 0 ? 0 : tr.tile_at(ps.first + pslice) * S::KT + lane * box) & ((1 << shift) - 1);
            const int64_t row = cell_row(page, ps.vhead, slot, a.c.kv_heads, shift);
            const uint64_t pol = l2_policy_evict_normal();
            constexpr int HALVES = S::ROW > 128 ? 2 : 1, W = S::ROW / HALVES;
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
                tma_load_2d(dst + h * (S::KT * W) + lane * box * W, &maps.k, h * 64, (int)row, bar, pol);
                tma_load_2d(dst + PART + h * (S::KT * W) + lane * box * W, &maps.v, h * 64, (int)row, bar, pol);
            }
            if (FMT != KV_FP16) {
                bulk_g2s(sdst + lane * box * 2, a.c.k_scale + row, box * 2, bar, pol);
                bulk_g2s(sdst + 128 + lane * box * 2, a.c.v_scale + row, box * 2, bar, pol);
            }
        }
        pslice += WARPS;
        ++issued;
    };
    for (int i = 0; i < STAGES; ++i) issue();

    int used = 0;
    bool dead = false;
    Segment sg;
    while (walk.next(a.s, w, &sg)) {
        // ---- the rows of the item: lane / 4 and lane / 4 + 8 ----
        const int p0 = sg.p0(w), p1 = sg.p1(w), lo0 = window_begin(p0 < 0 ? 0 : p0, w.window), lo1 = window_begin(p1 < 0 ? 0 : p1, w.window);
        const TileRange tr = sg.tiles(w);
        int row[2], head[2], pos[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = quad + 8 * h, t = sg.qt * w.tokens + r / w.group;
            const bool on = r < w.tokens * w.group && t < sg.n;
            row[h] = on ? sg.row0 + t : -1;
            head[h] = sg.vhead * w.group + r % w.group;
            pos[h] = on ? sg.len - sg.n + t : -1;
        }
        uint32_t q[D / 16][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t* src = reinterpret_cast<const uint32_t*>(a.q + (int64_t)(row[h] < 0 ? 0 : row[h]) * a.q_stride + (int64_t)head[h] * D);
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {   // fp16 cells: dims 2c, 2c + 1 and 8 behind; 8-bit cells: the four dims 4c .. that a word of codes holds
                uint2 x = make_uint2(0, 0);
                if (row[h] >= 0) x = FMT == KV_FP16 ? make_uint2(src[8 * k + c], src[8 * k + c + 4]) : *reinterpret_cast<const uint2*>(src + 8 * k + 2 * c);
                q[k][h] = x.x;
                q[k][2 + h] = x.y;
            }
        }
        State<D> st;
        st.clear();
        for (int slice = warp; slice < sg.count; slice += WARPS) {
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
            if (edge) {   // values that no row sees: whatever lies there, their weight is 0 and they must not be NaN
                for (int i = lane; i < S::KT * (S::ROW / 16); i += 32) {
                    const int r = i / (S::ROW / 16), key = k0 + r;
                    if (key > p1 || (key < lo0 && key >= w.sinks) || !(here >> (r >> box_shift) & 1u))
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(chunk_at<FMT, D>(vb, r, i % (S::ROW / 16))), "r"(0) : "memory");
                }
                __syncwarp();
            }
            float s[S::NT][4];
#pragma unroll
            for (int n = 0; n < S::NT; ++n) {
                s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
                for (int j = 0; j < S::ROW / 64; ++j) {   // four 16-byte pieces of 8 keys
                    uint32_t r[4];
                    ldsm_x4(chunk_at<FMT, D>(kb, n * 8 + (lane & 7), 4 * j + (lane >> 3)), r[0], r[1], r[2], r[3]);
                    if (FMT == KV_FP16) {
                        mma_16816(s[n], q[2 * j][0], q[2 * j][1], q[2 * j][2], q[2 * j][3], r[0], r[1]);
                        mma_16816(s[n], q[2 * j + 1][0], q[2 * j + 1][1], q[2 * j + 1][2], q[2 * j + 1][3], r[2], r[3]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            uint32_t b0, b1;
                            codes_to_half2x2<FMT>(r[i], b0, b1);
                            mma_16816(s[n], q[4 * j + i][0], q[4 * j + i][1], q[4 * j + i][2], q[4 * j + i][3], b0, b1);
                        }
                    }
                }
            }
            // scores as powers of two, with the scales of the two keys of this lane
            float inv[S::NT][2];
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < S::NT; ++n) {
                float ka = scale2, kc = scale2, ba = 0.f, bc = 0.f;
                if (FMT != KV_FP16) {
                    uint32_t ks, vs;
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(ks) : "r"(sb + (n * 8 + 2 * c) * 2));
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(vs) : "r"(sb + 128 + (n * 8 + 2 * c) * 2));
                    const float2 kf = half2_floats(ks), vf = half2_floats(vs);
                    ka = scale2 * kf.x;
                    kc = scale2 * kf.y;
                    ba = lg2(vf.x);
                    bc = lg2(vf.y);
                    inv[n][0] = ex2(-ba);
                    inv[n][1] = ex2(-bc);
                }
                s[n][0] = FMT == KV_FP16 ? s[n][0] * ka : fmaf(s[n][0], ka, ba);
                s[n][1] = FMT == KV_FP16 ? s[n][1] * kc : fmaf(s[n][1], kc, bc);
                s[n][2] = FMT == KV_FP16 ? s[n][2] * ka : fmaf(s[n][2], ka, ba);
                s[n][3] = FMT == KV_FP16 ? s[n][3] * kc : fmaf(s[n][3], kc, bc);
                if (edge) {
                    const int key = k0 + n * 8 + 2 * c;
                    const bool there = here >> ((n * 8) >> box_shift) & 1u;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!there || !key_visible(key + (i & 1), pos[i >> 1], w.window, w.sinks)) s[n][i] = -INFINITY;
                }
                top[0] = fmaxf(top[0], fmaxf(s[n][0], s[n][1]));
                top[1] = fmaxf(top[1], fmaxf(s[n][2], s[n][3]));
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
            }
            if (__any_sync(0xffffffffu, top[0] > st.m[0] || top[1] > st.m[1])) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float up = fmaxf(st.m[h], top[h]), f = st.m[h] == -INFINITY ? 0.f : ex2(st.m[h] - up);
                    st.m[h] = up;
                    st.l[h] *= f;
#pragma unroll
                    for (int i = 0; i < S::DT; ++i) {
                        st.o[i][2 * h] *= f;
                        st.o[i][2 * h + 1] *= f;
                    }
                }
            }
            const float ref[2] = {st.m[0] == -INFINITY ? 0.f : st.m[0], st.m[1] == -INFINITY ? 0.f : st.m[1]};
            uint32_t p[S::NT][2];
#pragma unroll
            for (int n = 0; n < S::NT; ++n) {
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    e[i] = ex2(s[n][i] - ref[i >> 1]);
                    if (FMT == KV_FP16) st.l[i >> 1] += e[i];
                    else if (!edge || s[n][i] != -INFINITY) st.l[i >> 1] = fmaf(e[i], inv[n][i & 1], st.l[i >> 1]);   // (the scale of a cell that is not there may be anything)
                }
                p[n][0] = floats_half2(e[0], e[1]);
                p[n][1] = floats_half2(e[2], e[3]);
            }
#pragma unroll
            for (int j = 0; j < S::KT / 16; ++j) {
                const uint32_t a0 = p[2 * j][0], a1 = p[2 * j][1], a2 = p[2 * j + 1][0], a3 = p[2 * j + 1][1];
#pragma unroll
                for (int d = 0; d < S::ROW / 32; ++d) {   // two 16-byte pieces of 16 keys
                    uint32_t r[4];
                    ldsm_x4_t(chunk_at<FMT, D>(vb, 16 * j + ((lane >> 3) & 1) * 8 + (lane & 7), 2 * d + (lane >> 4)), r[0], r[1], r[2], r[3]);
                    if (FMT == KV_FP16) {
                        mma_16816(st.o[2 * d], a0, a1, a2, a3, r[0], r[1]);
                        mma_16816(st.o[2 * d + 1], a0, a1, a2, a3, r[2], r[3]);
                    } else {
                        // a word holds dims 2 quad and 2 quad + 1 of two keys: one product for the even dims, one for the odd ones
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            uint32_t e0, o0, e1, o1;
                            codes_to_half2x2<FMT>(__byte_perm(r[2 * i], 0u, 0x3120), e0, o0);
                            codes_to_half2x2<FMT>(__byte_perm(r[2 * i + 1], 0u, 0x3120), e1, o1);
                            mma_16816(st.o[4 * d + 2 * i], a0, a1, a2, a3, e0, e1);
                            mma_16816(st.o[4 * d + 2 * i + 1], a0, a1, a2, a3, o0, o1);
                        }
                    }
                }
            }
            if (edge) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // (the zeros above, before a copy lands there)
            __syncwarp();
            if (!dead) issue();
        }

        // ---- the block's result of this segment, in warp 0 ----
        st.close();
        merge_warps<FMT, D>(st, smem + S_MERGE, warp, two);
        bool whole = sg.count == sg.total;
        if (!whole) {   // one of several blocks: the last to arrive adds the parts up, in the blocks' order
            const int b0 = (int)(sg.unit0 / chunk), b1 = (int)((sg.unit0 + sg.total - 1) / chunk);
            volatile int* flag = reinterpret_cast<volatile int*>(smem + S_FLAG);
            float4* parts = reinterpret_cast<float4*>(a.parts);
            if (warp == 0) {
                st.store(parts + (int64_t)(2 * blockIdx.x + (sg.first == 0 ? 1 : 0)) * (ATTN_DECODE_PART / 16), two);
                __threadfence();
                __syncwarp();
                if (lane == 0) {
                    const unsigned before = atomicAdd(a.counters + b0, 1u);
                    const bool last = before == (unsigned)(b1 - b0);
                    if (last) a.counters[b0] = 0u;
                    *flag = last;
                }
            }
            __syncthreads();
            whole = *flag != 0;
            if (whole) {
                __threadfence();
                st.clear();
                for (int b = b0 + warp; b <= b1; b += WARPS) st.add(parts + (int64_t)(2 * b + (b == b0 ? 1 : 0)) * (ATTN_DECODE_PART / 16), two);
                merge_warps<FMT, D>(st, smem + S_MERGE, warp, two);
            }
            __syncthreads();
        }
        if (whole && warp == 0) {
            unsigned again[2];   // rows that are not finite, or see nothing: from the formula once more, which does not touch hidden cells
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float f = 1.f / st.l[h];
                bool fine = st.l[h] > 0.f && st.l[h] < INFINITY;
#pragma unroll
                for (int i = 0; i < S::DT; ++i) {
                    st.o[i][2 * h] *= f;
                    st.o[i][2 * h + 1] *= f;
                    fine = fine && fabsf(st.o[i][2 * h]) < INFINITY && fabsf(st.o[i][2 * h + 1]) < INFINITY;
                }
                unsigned bad = __ballot_sync(0xffffffffu, !fine && row[h] >= 0);
                bad |= bad >> 1;
                bad |= bad >> 2;
                again[h] = bad & 0x11111111u;
                if (row[h] >= 0 && !(again[h] >> (lane & 28) & 1u)) {
                    uint32_t* out = reinterpret_cast<uint32_t*>(a.out + (int64_t)row[h] * a.o_stride + (int64_t)head[h] * D);
#pragma unroll
                    for (int i = 0; i < S::DT; ++i) {
                        if (FMT == KV_FP16) out[4 * i + c] = floats_half2(st.o[i][2 * h], st.o[i][2 * h + 1]);
                        else if (i % 2 == 0)   // dims 4c .. of 16: even, odd, even, odd
                            *reinterpret_cast<uint2*>(out + 4 * i + 2 * c) = make_uint2(floats_half2(st.o[i][2 * h], st.o[i + 1][2 * h]),
                                                                                      floats_half2(st.o[i][2 * h + 1], st.o[i + 1][2 * h + 1]));
                    }
                }
            }
#pragma unroll 1
            for (int h = 0; h < 2; ++h)
                for (unsigned left = again[h]; left; left &= left - 1) {
                    const int from = __ffs(left) - 1;
                    const int r = __shfl_sync(0xffffffffu, row[h], from), hd = __shfl_sync(0xffffffffu, head[h], from), ps2 = __shfl_sync(0xffffffffu, pos[h], from);
                    if (!attend_row<FMT, D>(a, sg.seq, sg.len, ps2, r, hd) && lane == 0) *a.status = STATUS_BAD_TABLE;
                }
        }
    }
    // (after a wait that ran out: what was asked for must land before the block's memory is given back)
    if (dead)
        for (int i = issued < STAGES ? 0 : issued - STAGES; i < issued; ++i) mbar_wait_bounded_warp(bars + (i % STAGES) * 8, (i / STAGES) & 1);
}

}  // namespace

cudaError_t attention_decode_configure() {
    cudaError_t e = cudaSuccess;
    auto one = [&](auto* k) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    };
    one(attention_decode_kernel<KV_FP16, 64>);
    one(attention_decode_kernel<KV_FP16, 128>);
    one(attention_decode_kernel<KV_INT8, 64>);
    one(attention_decode_kernel<KV_INT8, 128>);
    one(attention_decode_kernel<KV_FP8, 64>);
    one(attention_decode_kernel<KV_FP8, 128>);
    return e;
}

int attention_decode_keys(int fmt, int dim) { return PART / (dim * kv_cell_bytes(fmt)); }

cudaError_t launch_attention_decode(const AttnArgs& a, const AttnMaps& maps, int sm_count, cudaStream_t st, bool pdl) {
    auto k = a.c.fmt == KV_FP16 ? (a.c.dim == 64 ? attention_decode_kernel<KV_FP16, 64> : attention_decode_kernel<KV_FP16, 128>)
             : a.c.fmt == KV_INT8 ? (a.c.dim == 64 ? attention_decode_kernel<KV_INT8, 64> : attention_decode_kernel<KV_INT8, 128>)
                                  : (a.c.dim == 64 ? attention_decode_kernel<KV_FP8, 64> : attention_decode_kernel<KV_FP8, 128>);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(sm_count < ATTN_MAX_BLOCKS ? sm_count : ATTN_MAX_BLOCKS));
    cfg.blockDim = dim3(WARPS * 32);
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
