// Attention of many query rows to a cache head (chunks of new tokens, prompts, drafts): two products on the tensor cores per tile of keys.
//
//   t_k = scale log2(e) q.k,  w_k = 2^(t_k - m),  out = sum w_k v_k / sum w_k       m: a running reference, 7 to 15 below the maximum of t
//
// (8-bit cells: the scales join the scores and weights as in attention_decode.cu: codes are exact in fp16, no rounding is added.  Weights up to 2^15 for
// the reason given there.)
//
// An item is up to 256 query rows: two tiles of 128, each new tokens times the query heads of a cache head, so that a cell is
// fetched once for all heads that share it.  With no more than 128 rows the two tiles hold the same rows and take the key tiles in turn.
// A block is one of each SM:
//   * warps 0-7 and 8-15: the softmax of one query tile each, two threads per row, 64 keys each (one thread per row left two warps to a
//     scheduler, which were idle half of the time on each other's latencies: 3500 clocks for a pair of tiles of 64 dims, 2800 here): scores come
//     from tensor memory and stay in registers, the weights go back there as fp16 in the scores' place (the A operand of the second product).  The
//     sums of outputs stay in tensor memory and are scaled again only when a row's maximum has grown by more than 2^8.
//   * warp 16: issues all tcgen05.mma: scores = Q K^T (both K-major), out += weights V (V as it lies in the cache, MN-major).  While one
//     query tile is in its softmax the other one has the tensor cores.
//   * warp 17: tensor copies (fp16: straight into the operands; 8-bit: codes into a ring of parts of tiles).
//   * warps 18 and 19 (cells of 128 dims: 20-23), 8-bit cells only: codes to fp16 operands, and the keys' factors.
// What bounds it: two tiles of 128 x 128 scores take 2048 clocks of the SM's exponential units and 16 D of its tensor cores; they take 2800 (fp16 of 64
// dims), 3240 (of 128) and with codes 3900 and 4700 to 4800, since a query tile's products wait for its softmax and the softmax for its scores.  2048 tokens of
// 32 heads to 8, to 16384 positions: fp16 of 64 dims 352 us (730 TFLOP/s; the exponentials alone some 235), of 128 dims 447 us (1150 TFLOP/s).
// 8-bit cells (64 dims 442 to 447, 128 dims 607 to 610 us) are bound by what expands them: codes go through shared memory twice, and the factors of
// 128 keys are read from there by every row.  An item costs 7500 clocks besides its keys (128 dims: 15500), of which 2400 (5400) are waits for its last products: the
// warps that store its result begin the next softmax.
#include <type_traits>

#include "attention_maps.h"
#include "attention_row.cuh"
#include "attention_work.cuh"
#include "tcgen05.cuh"

namespace nnb {
namespace {

constexpr int BN = 128;   // keys of a tile

// Where a warp is in its block's work.  It lies in shared memory: two dozen registers less in the softmax's loops.
struct Steps {
    Walk walk, begin;
    Segment sg, next;   // (the softmax warps fetch the next one's queries early)
};

template <int FMT, int D>
struct Chunk {
    static constexpr bool CODES = FMT != KV_FP16;
    static constexpr int HALVES = D / 64;                        // 128-byte columns of an operand tile
    static constexpr int TILE = BN * D * 2;                      // bytes of an operand tile
    static constexpr int RING = D == 64 ? 4 : 2;                 // key tiles, and as many value tiles
    // What the softmax needs of a key tile outlives the tile: tile t goes in when the products of tile t - RING are done, and then the softmax
    // of tile t - RING - 2 is.  (Its copies begin up to two tiles earlier.)
    static constexpr int META = D == 64 ? 8 : 4;
    static constexpr int HERE = 8;                               // which keys of a tile were copied: noted when its copies begin
    static constexpr int RAW_KEYS = 32, RAW = RAW_KEYS * D;      // codes arrive in parts of a tile, one for each expanding warp
    static constexpr int RAW_STAGE = RAW + 4 * RAW_KEYS;         // with the scales of keys and values
    static constexpr int RAWS = CODES ? (D == 64 ? 12 : 4) : 0; // a stage is always the same warp's: whose turn it is shows in one bit
    static constexpr int EXPANDERS = D == 64 ? 2 : 4;            // warps that expand codes
    static constexpr int FIRST_EXPANDER = EXPANDERS == 2 ? 18 : 20, THREADS = CODES && EXPANDERS == 4 ? 768 : 640;
    // shared memory
    static constexpr int O_Q = 0, O_K = O_Q + 2 * TILE, O_V = O_K + RING * TILE, O_RAW = O_V + RING * TILE, O_META = O_RAW + RAWS * RAW_STAGE;
    static constexpr int META_BYTES = CODES ? BN * 12 : 0;       // factors of the scores, their summands, 1 / scale of the values
    static constexpr int O_HERE = O_META + META * META_BYTES, O_SUMS = O_HERE + HERE * 4, O_WALK = O_SUMS + 5 * BN * 4, O_BARS = O_WALK + THREADS / 32 * (int)sizeof(Steps);
    static constexpr int B_KFULL = 0, B_KEMPTY = B_KFULL + RING, B_VFULL = B_KEMPTY + RING, B_VEMPTY = B_VFULL + RING, B_META = B_VEMPTY + RING,
                         B_RFULL = B_META + META, B_REMPTY = B_RFULL + RAWS, B_Q = B_REMPTY + RAWS, B_S = B_Q + 2, B_P = B_S + 2, B_O = B_P + 2, B_FIX = B_O + 2, B_DONE = B_FIX + 1,
                         BARS = B_DONE + 1;
    static constexpr int O_TMEM = O_BARS + BARS * 8, O_DEAD = O_TMEM + 4, BYTES = O_DEAD + 12, SMEM = BYTES + 1024;
    static_assert(SMEM <= 227 * 1024, "shared memory");
    static_assert(RAWS % (BN / RAW_KEYS) == 0, "a stage belongs to one part of a tile");
    static_assert(O_BARS % 8 == 0 && O_RAW % 128 == 0 && RAW_STAGE % 16 == 0 && O_META % 16 == 0, "alignment");
};
constexpr int T_S = 0, T_O = 256;   // tensor memory: two tiles of scores (and weights), two of outputs

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
// 32 columns of this thread's lane; the registers are valid after tmem_wait_ld32.
__device__ __forceinline__ void tmem_ld32_begin(uint32_t taddr, uint32_t (&u)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]),
          "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]),
          "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld32(uint32_t (&u)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]), "+r"(u[8]), "+r"(u[9]), "+r"(u[10]), "+r"(u[11]),
                   "+r"(u[12]), "+r"(u[13]), "+r"(u[14]), "+r"(u[15]), "+r"(u[16]), "+r"(u[17]), "+r"(u[18]), "+r"(u[19]), "+r"(u[20]), "+r"(u[21]), "+r"(u[22]),
                   "+r"(u[23]), "+r"(u[24]), "+r"(u[25]), "+r"(u[26]), "+r"(u[27]), "+r"(u[28]), "+r"(u[29]), "+r"(u[30]), "+r"(u[31])
                 :: "memory");
}
// Two 32-bit values in one instruction
__device__ __forceinline__ uint64_t pair(uint32_t a, uint32_t b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint64_t pair(float a, float b) { return pair(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ void unpair(uint64_t d, uint32_t& a, uint32_t& b) { asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(d)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
template <int N>
__device__ __forceinline__ void set_registers_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void set_registers_fewer() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// Bits [0, n) of 32
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }

// An operand whose N dimension lies together (V: dims of a key): tiles of 64 dims x 8 keys; the leading offset is the distance of
// two 64-dim columns, the stride that of two groups of 8 keys (1024 bytes).
__device__ __forceinline__ uint32_t desc_lo_mn(uint32_t saddr, uint32_t column_bytes) { return ((saddr >> 4) & 0x3FFFu) | ((column_bytes >> 4) << 16); }
constexpr uint32_t IDESC_B_MN = 1u << 16;

__device__ __forceinline__ void st_shared16(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// 16 bytes `chunk` of row `row` of an operand tile
__device__ __forceinline__ uint32_t operand_at(uint32_t tile, int row, int chunk) {
    return tile + (chunk >> 3) * (BN * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

// What an item's rows are: query tile i (0 or 1) holds tokens [first(i), last(i)] of the sequence.
struct ItemRows {
    int t0, t1;       // tokens of the item
    int per;          // tokens of a query tile
    bool turns;       // both query tiles hold the same rows
    __device__ __forceinline__ ItemRows(const Segment& s, const WorkShape& w) {
        t0 = s.qt * w.tokens;
        t1 = min(t0 + w.tokens, s.n) - 1;
        per = w.tokens / 2;
        turns = t1 - t0 + 1 <= per;
    }
    __device__ __forceinline__ int first(int i) const { return turns ? t0 : t0 + i * per; }
    __device__ __forceinline__ int last(int i) const { return turns ? t1 : min(t1, t0 + (i + 1) * per - 1); }
};

// Two warps (named barrier `id`): wait for each other; and whether any of their threads says yes.
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool pair_any(int id, bool yes) {
    int r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, 64, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((int)yes), "r"(id) : "memory");
    return r != 0;
}

__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 9, 512;" ::: "memory"); }

// The 512 threads of the softmax, after their part of an item that several blocks share has been written: where it is the last one to
// arrive, adds all of them up, in the blocks' order.  True: some row of this thread's is not finite (it is marked).
template <int D>
__device__ __forceinline__ bool join_parts(const AttnArgs& a, const Segment& sg, const WorkShape& w, const ItemRows& rows, int parts, volatile int* joined) {
    const int tid = threadIdx.x, b0 = (int)(sg.unit0 / w.chunk), b1 = (int)((sg.unit0 + sg.total - 1) / w.chunk), id = sg.first ? 1 : 2;
    __threadfence();
    softmax_sync();
    if (tid == 0) {
        const bool last = atomicAdd(a.counters + b0, 1u) == (unsigned)(b1 - b0);
        if (last) {
            a.counters[b0] = 0u;
            *joined = *joined | id;
        }
    }
    softmax_sync();
    if (!(*joined & id)) return false;
    __threadfence();
    // a row to a thread, and half of its dims, or a quarter where there are 128 rows
    const int r = rows.turns ? tid & 127 : tid & 255, i = r >> 7, rr = r & 127, t = rows.first(i) + rr / w.group, hg = (sg.vhead % parts) * w.group + rr % w.group;
    const bool on = rr < rows.per * w.group && t <= rows.last(i) && hg < a.group;
    const int quads = rows.turns ? D / 16 : D / 8, q0 = (rows.turns ? tid >> 7 : tid >> 8) * quads;
    const float4* base = reinterpret_cast<const float4*>(a.parts);
    auto part = [&](int b) { return base + (int64_t)(2 * b + (b == b0 ? 1 : 0)) * (ATTN_CHUNK_PART / 16); };
    auto sums = [&](int b) { return reinterpret_cast<const float2*>(part(b) + 64 * D)[r]; };   // maximum and sum of the weights
    float m = -INFINITY, l = 0.f;
#pragma unroll 4
    for (int b = b0; b <= b1; ++b) m = fmaxf(m, sums(b).x);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll 4
    for (int b = b0; b <= b1; ++b) {
        const float2 x = sums(b);
        l = fmaf(x.y, ex2(x.x - ref), l);
    }
    const float inv = 1.f / l;
    bool fine = l > 0.f && l < INFINITY;
    uint16_t* const out = a.out + (int64_t)(sg.row0 + t) * a.o_stride + (int64_t)(sg.vhead / parts * a.group + hg) * D;
#pragma unroll 1
    for (int q = q0; q < q0 + quads; q += 4) {
        float4 o[4] = {};
#pragma unroll 2
        for (int b = b0; b <= b1; ++b) {
            const float4* p = part(b) + q * 256 + r;
            float4 v[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) v[x] = p[x * 256];
            const float f = ex2(sums(b).x - ref);
#pragma unroll
            for (int x = 0; x < 4; ++x) o[x] = make_float4(fmaf(v[x].x, f, o[x].x), fmaf(v[x].y, f, o[x].y), fmaf(v[x].z, f, o[x].z), fmaf(v[x].w, f, o[x].w));
        }
        uint32_t h[8];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const float y[4] = {o[x].x * inv, o[x].y * inv, o[x].z * inv, o[x].w * inv};
            fine = fine && fabsf(y[0]) < HALF_END && fabsf(y[1]) < HALF_END && fabsf(y[2]) < HALF_END && fabsf(y[3]) < HALF_END;
            h[2 * x] = floats_half2(y[0], y[1]);
            h[2 * x + 1] = floats_half2(y[2], y[3]);
        }
        if (on) {
            reinterpret_cast<uint4*>(out + 4 * q)[0] = make_uint4(h[0], h[1], h[2], h[3]);
            reinterpret_cast<uint4*>(out + 4 * q)[1] = make_uint4(h[4], h[5], h[6], h[7]);
        }
    }
    softmax_sync();
    if (on && !fine) *out = 0x7FFF;
    return on && !fine;
}

template <int FMT, int D, bool TREE>
__global__ void __launch_bounds__(Chunk<FMT, D>::THREADS, 1) attention_chunk_kernel(const __grid_constant__ AttnMaps maps, const AttnArgs a) {
    using C = Chunk<FMT, D>;
    constexpr int RAWS = C::CODES ? C::RAWS : 1;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t base = smem_u32(smem), bars = base + C::O_BARS;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    auto bar = [&](int i) { return bars + (uint32_t)i * 8; };
    volatile int* dead = reinterpret_cast<volatile int*>(smem + C::O_DEAD);
    volatile int* some_again = dead + 1;   // some row of the items that the block has finished has to be computed once more
    volatile int* joined = dead + 2;       // which of its parts of items the block has joined with the others: 1 its first one, 2 its last one
    // Waits of whole warps.  When one runs out the block carries on without waiting: what it computes is void, and ends.
    auto wait = [&](int b, uint32_t parity) {
        uint32_t ok = mbar_try_wait(bar(b), parity);
        if (__all_sync(0xffffffffu, ok)) return;
        const long long t0 = clock64();
        for (;;) {
            if (!ok) ok = mbar_try_wait(bar(b), parity);
            if (__all_sync(0xffffffffu, ok)) return;
            if (__any_sync(0xffffffffu, *dead || clock64() - t0 > WAIT_CYCLES)) {
                *dead = 1;
                *a.status = 32;
                return;
            }
        }
    };
    auto given_up = [&]() { return __any_sync(0xffffffffu, *dead) != 0; };
    if (tid < C::BARS) {
        const int b = tid;
        int n = 1;
        if (b < C::B_KEMPTY || (b >= C::B_VFULL && b < C::B_VEMPTY) || (b >= C::B_META && b < C::B_RFULL)) n = C::CODES ? C::EXPANDERS : 1;
        if ((b >= C::B_Q && b < C::B_S) || (b >= C::B_P && b < C::B_O)) n = 8;
        mbar_init(bar(b), n);
    }
    if (tid == 0) *dead = *some_again = *joined = 0;
    mbar_init_fence();
    if (warp == 16) tmem_alloc<false>(base + C::O_TMEM, 512);
    tc_fence_before();
    pdl_wait_prior_grid();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + C::O_TMEM);

    WorkShape w;
    const int parts = (a.group + 127) / 128;   // parts of a cache head's query heads
    w.group = (a.group + parts - 1) / parts;
    w.tokens = 2 * (128 / w.group);
    w.vheads = a.c.kv_heads * parts;
    w.tile = BN;
    w.window = a.window;
    w.sinks = a.sinks;
    w.tree_words = TREE ? a.tree_words : 0;
    w.extra = ATTN_CHUNK_EXTRA;
    w.second = TREE ? 2 * ATTN_CHUNK_EXTRA : 0;   // (other calls keep the order of sums that they have had)
    Steps& steps = reinterpret_cast<Steps*>(smem + C::O_WALK)[warp];
    Segment& sg = steps.sg;
    {
        const Walk walk = find_work(a.s, &w, 2, a.status);
        if (lane == 0) steps.walk = steps.begin = walk;
    }
    auto next_into = [&](Segment* to) {
        int more = 0;
        __syncwarp();
        if (lane == 0) more = steps.walk.next(a.s, w, to);
        __syncwarp();   // (the other lanes read the segment next: a shuffle orders registers alone)
        return __shfl_sync(0xffffffffu, more, 0) != 0;
    };
    auto next_segment = [&]() { return next_into(&steps.sg); };
    const int shift = a.c.page_shift;
    const float scale2 = a.scale * 1.4426950408889634f;
    int4* const info = a.items + blockIdx.x;   // for the kernel that joins the parts: what this block has begun and not finished
    if (tid == 0 && !a.join_here) *info = make_int4(-1, 0, 0, 0);

    // Registers of a thread: more for the four groups of four warps that do the softmax, fewer for the others.  The shares add up to what the block
    // was launched with: 4 x 104 + 64 = 5 x 96, 4 x 96 + 2 x 48 = 6 x 80.  (With 88 and 64 of the latter int8 cells, 2048 tokens of 32 heads of 128 dims to
    // 16384 positions, took 734 us instead of 684.)
    if (warp < 16) set_registers_more<C::THREADS == 640 ? 104 : 96>();
    else set_registers_fewer<C::THREADS == 640 ? 64 : 48>();
    if (warp < 16) {
        // ---- softmax of query tile i, keys 64 c .. of a tile; row r ----
        const int i = warp >> 3, c = warp >> 2 & 1, r = tid & 127, pair_bar = 1 + i * 4 + (warp & 3);
        // What the threads of a row tell each other: [tile][half of the keys][row], and behind it the references of the second tile.
        volatile float* const said = reinterpret_cast<volatile float*>(smem + C::O_SUMS) + r;
        volatile float *const other = said + (i * 2 + (c ^ 1)) * BN, *const own = said + (i * 2 + c) * BN;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, ts = tmem + T_S + i * BN + c * 64 + lanes, to = tmem + T_O + i * D + c * (D / 2) + lanes;
        const uint32_t qtile = base + C::O_Q + i * C::TILE;
        uint32_t s_phase = 0, o_phase = 0;
        int kt = 0;   // key tiles of the block so far
        // This thread's half of its row of a segment's queries, to where the products take them from.
        auto queries = [&](const Segment& s) {
            const ItemRows rows(s, w);
            const int kv_head = s.vhead / parts, g = r % w.group, t = rows.first(i) + r / w.group, hg = (s.vhead % parts) * w.group + g;
            const bool on = r < rows.per * w.group && t <= rows.last(i) && hg < a.group;
            const uint4* src = reinterpret_cast<const uint4*>(a.q + (int64_t)(s.row0 + t) * a.q_stride + (int64_t)(kv_head * a.group + hg) * D) + c * (D / 16);
            uint4 v[D / 16];
#pragma unroll
            for (int x = 0; x < D / 16; ++x) v[x] = on ? src[x] : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int x = 0; x < D / 16; ++x) st_shared16(operand_at(qtile, r, c * (D / 16) + x), v[x]);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(C::B_Q + i));
        };
        bool more = next_segment();
        if (more) queries(sg);
        while (more) {
            const ItemRows rows(sg, w);
            const TileRange tr = sg.tiles(w);
            const int kv_head = sg.vhead / parts, g = r % w.group, t = rows.first(i) + r / w.group, hg = (sg.vhead % parts) * w.group + g;
            const bool on = r < rows.per * w.group && t <= rows.last(i) && hg < a.group;
            const int row = sg.row0 + t, head = kv_head * a.group + hg, pos = on ? sg.len - sg.n + t : -1, lo = window_begin(pos < 0 ? 0 : pos, w.window);
            // positions of the tile's first and last token
            const int pmin = TREE ? sg.p0(w) : sg.len - sg.n + rows.first(i), pmax = sg.len - sg.n + rows.last(i), lo_max = window_begin(pmax < 0 ? 0 : pmax, w.window);
            float m = -INFINITY, l = 0.f;
            bool first = true;
            for (int j = rows.turns ? i : 0; j < sg.count; j += rows.turns ? 2 : 1) {
                const int mt = (kt + j) % C::META;
                wait(C::B_META + mt, ((kt + j) / C::META) & 1);
                wait(C::B_S + i, s_phase);
                s_phase ^= 1;
                tc_fence_after();
                const int k0 = sg.p1(w) < 0 ? 0 : tr.tile_at(sg.first + j) * BN;
                const unsigned here = *reinterpret_cast<volatile unsigned*>(smem + C::O_HERE + (kt + j) % C::HERE * 4);
                const bool edge = here != 0xFFu || k0 + BN - 1 > pmin || (k0 < lo_max && k0 + BN > w.sinks);
                const float4* fa = reinterpret_cast<const float4*>(smem + C::O_META + mt * C::META_BYTES) + c * 16;   // factors of four keys' scores
                const float4 *fb = fa + BN / 4, *inv = fb + BN / 4;                                                  // their summands; 1 / scale of the values
                uint32_t v[2][32];
                tmem_ld32_begin(ts, v[0]);
                tmem_ld32_begin(ts + 32, v[1]);
                // Scores as powers of two (fp16: times 1 / scale2 still), -infinity where the row does not see the key; their maximum.
                float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
                for (int cb = 0; cb < 2; ++cb) {
                    tmem_wait_ld32(v[cb]);
                    if (C::CODES) {
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            const float4 f = fa[cb * 8 + x], b = fb[cb * 8 + x];
                            unpair(fma2(pair(v[cb][4 * x], v[cb][4 * x + 1]), pair(f.x, f.y), pair(b.x, b.y)), v[cb][4 * x], v[cb][4 * x + 1]);
                            unpair(fma2(pair(v[cb][4 * x + 2], v[cb][4 * x + 3]), pair(f.z, f.w), pair(b.z, b.w)), v[cb][4 * x + 2], v[cb][4 * x + 3]);
                        }
                    }
                    if (edge) {
                        const int at = k0 + c * 64 + cb * 32;
                        uint32_t seen;
                        if (TREE) seen = on ? tree_bits(a.tree + (int64_t)row * a.tree_words, a.tree_words, at, sg.len - sg.n, sg.len) : 0u;
                        else seen = low_bits(pos + 1 - at) & (~low_bits(lo - at) | low_bits(w.sinks - at));
                        const unsigned there = here >> (4 * c + 2 * cb);
                        seen &= ((there & 1u) ? 0xFFFFu : 0u) | ((there & 2u) ? 0xFFFF0000u : 0u);
#pragma unroll
                        for (int x = 0; x < 32; ++x)
                            if (!(seen >> x & 1u)) v[cb][x] = 0xFF800000u;
                    }
#pragma unroll
                    for (int x = 0; x < 32; x += 4) {
                        t0 = max3(t0, __uint_as_float(v[cb][x]), __uint_as_float(v[cb][x + 1]));
                        t1 = max3(t1, __uint_as_float(v[cb][x + 2]), __uint_as_float(v[cb][x + 3]));
                    }
                }
                float top = fmaxf(t0, t1);
                if (!C::CODES) top *= scale2;
                // Both threads of a row keep the same reference: they agree whether some row of their two warps wants another one.
                if (pair_any(pair_bar, first || top - m > 15.f)) {
                    *own = top;
                    pair_sync(pair_bar);
                    const float up = fmaxf(m, fmaxf(top, *other) - 7.f), f = m == -INFINITY ? 0.f : ex2(m - up);
                    m = up;
                    if (!first) {   // (the scores came after the product before, so the sums are complete)
                        l *= f;
#pragma unroll 1
                        for (int cb = 0; cb < D / 32; ++cb) {
                            uint32_t o[16];
                            tmem_ld16(to + cb * 16, o);
#pragma unroll
                            for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                            tmem_st16(to + cb * 16, o);
                        }
                        tmem_wait_st();
                    }
                }
                first = false;
                // the weights
                const float ref = m == -INFINITY ? 0.f : -m;
                const uint64_t ref2 = pair(ref, ref), mul2 = pair(scale2, scale2);
                uint64_t sum2[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
                for (int cb = 0; cb < 2; ++cb) {
                    uint32_t p[16];
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        float e[4];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint64_t sc = pair(v[cb][4 * x + 2 * h], v[cb][4 * x + 2 * h + 1]);
                            uint32_t u0, u1;
                            unpair(C::CODES ? add2(sc, ref2) : fma2(sc, mul2, ref2), u0, u1);
                            e[2 * h] = ex2(__uint_as_float(u0));
                            e[2 * h + 1] = ex2(__uint_as_float(u1));
                        }
                        if (C::CODES) {
                            const float4 n = inv[cb * 8 + x];
                            sum2[0] = fma2(pair(e[0], e[1]), pair(n.x, n.y), sum2[0]);
                            sum2[1] = fma2(pair(e[2], e[3]), pair(n.z, n.w), sum2[1]);
                        } else {
                            sum2[0] = add2(sum2[0], pair(e[0], e[1]));
                            sum2[1] = add2(sum2[1], pair(e[2], e[3]));
                        }
                        p[2 * x] = floats_half2(e[0], e[1]);
                        p[2 * x + 1] = floats_half2(e[2], e[3]);
                    }
                    tmem_st16(ts + cb * 16, p);
                }
                {
                    uint32_t u0, u1;
                    unpair(add2(sum2[0], sum2[1]), u0, u1);
                    l += __uint_as_float(u0) + __uint_as_float(u1);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(C::B_P + i));
            }
            kt += sg.count;

            // ---- the segment's result ----
            const bool mine = rows.turns ? i < sg.count : true;   // this tile has had keys
            // The next segment's queries: the products have taken this one's, as the scores of its last tile have come, and go on meanwhile.
            more = next_into(&steps.next);
            if (more && mine) queries(steps.next);
            if (mine) {
                wait(C::B_O + i, o_phase);
                o_phase ^= 1;
            }
            float f0 = 1.f, f1 = 0.f;   // factors of this tile's sums and, where the tiles take turns, of the other's
            *own = l;
            if (rows.turns && i == 1) said[4 * BN] = m;
            if (rows.turns) softmax_sync();
            else pair_sync(pair_bar);
            l += *other;
            if (rows.turns && i == 0) {
                const float m1 = said[4 * BN], up = fmaxf(m, m1);
                f0 = m == -INFINITY ? 0.f : ex2(m - up);
                f1 = m1 == -INFINITY ? 0.f : ex2(m1 - up);
                l = l * f0 + (said[2 * BN] + said[3 * BN]) * f1;
                m = up;
            }
            tc_fence_after();
            if (i == 0 || !rows.turns) {
                const bool both = rows.turns && sg.count > 1, whole = sg.count == sg.total;
                const float scale_out = whole ? 1.f / l : 1.f;
                float4* part = reinterpret_cast<float4*>(a.parts) + (int64_t)(2 * blockIdx.x + (sg.first == 0 ? 1 : 0)) * (ATTN_CHUNK_PART / 16);
                uint16_t* out = a.out + (int64_t)row * a.o_stride + (int64_t)head * D + c * (D / 2);
                bool fine = l > 0.f && l < INFINITY;
#pragma unroll 1
                for (int cb = 0; cb < D / 32; ++cb) {
                    uint32_t o[16];
                    float v[16];
                    tmem_ld16(to + cb * 16, o);
#pragma unroll
                    for (int x = 0; x < 16; ++x) v[x] = __uint_as_float(o[x]) * f0;
                    if (both) {
                        tmem_ld16(to + D + cb * 16, o);
#pragma unroll
                        for (int x = 0; x < 16; ++x) v[x] = fmaf(__uint_as_float(o[x]), f1, v[x]);
                    }
                    if (!whole) {
#pragma unroll
                        for (int x = 0; x < 4; ++x) part[(c * (D / 8) + cb * 4 + x) * 256 + i * 128 + r] = make_float4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]);
                        continue;
                    }
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        v[x] *= scale_out;
                        fine = fine && fabsf(v[x]) < HALF_END;
                    }
                    if (on) {
#pragma unroll
                        for (int x = 0; x < 2; ++x)
                            reinterpret_cast<uint4*>(out)[cb * 2 + x] = make_uint4(floats_half2(v[8 * x], v[8 * x + 1]), floats_half2(v[8 * x + 2], v[8 * x + 3]),
                                                                                  floats_half2(v[8 * x + 4], v[8 * x + 5]), floats_half2(v[8 * x + 6], v[8 * x + 7]));
                    }
                }
                if (!whole) {
                    if (c == 0) reinterpret_cast<float2*>(part + 64 * D)[i * 128 + r] = make_float2(m, l);
                    if (!a.join_here && sg.first == 0 && tid == 0) *info = make_int4(sg.seq, sg.vhead, sg.qt, (int)((sg.unit0 + sg.total - 1) / w.chunk));
                } else {
                    // rows that are not finite in either half, or see nothing, are marked by a NaN
                    pair_sync(pair_bar);   // (the sums have been read)
                    *own = fine ? 0.f : 1.f;
                    pair_sync(pair_bar);
                    fine = fine && *other == 0.f;
                    if (c == 0 && on && !fine) {
                        *out = 0x7FFF;
                        *some_again = 1;
                    }
                }
            }
            if (a.join_here && sg.count != sg.total && join_parts<D>(a, sg, w, rows, parts, joined)) *some_again = 1;
            tc_fence_before();
            // (what the threads have told each other has been read)
            if (rows.turns) softmax_sync();
            else pair_sync(pair_bar);
            // (without keys of its own, this tile's barrier must not get two segments ahead of the products)
            if (more && !mine) queries(steps.next);
            __syncwarp();
            if (lane == 0) sg = steps.next;
            __syncwarp();
        }
        // Marked rows: from the formula once more, which does not use hidden cells.  Behind the loop: no wait of another warp runs out meanwhile, and
        // this takes no registers from it (int8 cells of 128 dims, 2048 tokens of 32 heads to 16384 positions: 675 us, 800 with this inside).
        softmax_sync();
        if (!*some_again) {
            // Not earlier: waits of the next launch have a limit, which counts from its beginning, and this kernel may run for longer than that.
            pdl_launch_dependents();
        } else {
            __syncwarp();
            if (lane == 0) steps.walk = steps.begin;
            while (next_segment()) {
                if (sg.count != sg.total && !(*joined & (sg.first ? 1 : 2))) continue;
                const ItemRows rows(sg, w);
                const int kv_head = sg.vhead / parts, x = warp >> 1, rr = (x & 3) * 32 + lane, g = rr % w.group, t = rows.first(x >> 2) + rr / w.group;
                const int hg = (sg.vhead % parts) * w.group + g, row = sg.row0 + t, head = kv_head * a.group + hg, pos = sg.len - sg.n + (TREE ? 0 : t);
                const bool on = !(rows.turns && x >= 4) && rr < rows.per * w.group && t <= rows.last(x >> 2) && hg < a.group;
                const bool marked = on && (*reinterpret_cast<const volatile uint16_t*>(a.out + (int64_t)row * a.o_stride + (int64_t)head * D) & 0x7FFF) > 0x7C00;
                for (unsigned left = __ballot_sync(0xffffffffu, marked) & (warp & 1 ? 0xAAAAAAAAu : 0x55555555u); left; left &= left - 1) {
                    const int from = __ffs(left) - 1;
                    const int r2 = __shfl_sync(0xffffffffu, row, from), h2 = __shfl_sync(0xffffffffu, head, from), p2 = __shfl_sync(0xffffffffu, pos, from);
                    if (!attend_row<FMT, D, TREE>(a, sg.seq, sg.len, p2, r2, h2) && lane == 0) a.status[STATUS_BAD_TABLE] = 1;
                }
            }
        }
    } else if (warp == 16) {
        // ---- products ----
        const bool issuer = elect_one();
        const uint32_t id_s = instr_desc_f16(BN, 128), id_o = instr_desc_f16(D, 128) | IDESC_B_MN;
        int kt = 0;
        uint32_t q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
        while (next_segment()) {
            const bool turns = ItemRows(sg, w).turns;
            const int n = sg.count;
            auto second = [&](int i, int j) {   // out += weights V of tile j
                const int slot = (kt + j) % C::RING;
                if (turns || i == 0) wait(C::B_VFULL + slot, ((kt + j) / C::RING) & 1);
                wait(C::B_P + i, p_phase[i]);
                p_phase[i] ^= 1;
                tc_fence_after();
                if (issuer) {
                    const uint32_t lo = desc_lo_mn(base + C::O_V + slot * C::TILE, BN * 128), ts = tmem + T_S + i * BN, to = tmem + T_O + i * D;
                    const bool begin = turns ? j == i : j == 0;
#pragma unroll
                    for (int k = 0; k < BN / 16; ++k) umma_f16_ts<false>(to, ts + (k >> 2) * 64 + (k & 3) * 8, desc_of(lo + k * 128), id_o, !(begin && k == 0));
                    if (turns || i == 1) umma_commit<false>(bar(C::B_VEMPTY + slot));
                }
                __syncwarp();
            };
            for (int v = 0; v < (turns ? n : 2 * n); ++v) {
                const int j = turns ? v : v >> 1, i = v & 1, before = turns ? j - 2 : j - 1;
                const int slot = (kt + j) % C::RING;
                if (turns || i == 0) wait(C::B_KFULL + slot, ((kt + j) / C::RING) & 1);
                if (before >= 0) second(i, before);
                if (before < 0) {
                    wait(C::B_Q + i, q_phase[i]);
                    q_phase[i] ^= 1;
                }
                tc_fence_after();
                if (issuer) {
                    const uint32_t qa = smem_desc_lo(base + C::O_Q + i * C::TILE), kb = smem_desc_lo(base + C::O_K + slot * C::TILE), ts = tmem + T_S + i * BN;
#pragma unroll
                    for (int k = 0; k < D / 16; ++k) {
                        const uint32_t at = (k >> 2) * (BN * 128 / 16) + (k & 3) * 2;
                        umma_f16<false>(ts, desc_of(qa + at), desc_of(kb + at), id_s, k > 0);
                    }
                    umma_commit<false>(bar(C::B_S + i));
                    if (turns || i == 1) umma_commit<false>(bar(C::B_KEMPTY + slot));
                }
                __syncwarp();
            }
            if (turns && n == 1) {   // the second query tile has no keys: its queries' barrier moves on all the same
                wait(C::B_Q + 1, q_phase[1]);
                q_phase[1] ^= 1;
            }
            for (int e = 0; e < (turns && n == 1 ? 1 : 2); ++e) {   // what is still out, in the order of the values
                const int tile = turns ? max(n - 2, 0) + e : n - 1, i = turns ? tile & 1 : e;
                second(i, tile);
                if (issuer) umma_commit<false>(bar(C::B_O + i));
                __syncwarp();
            }
            kt += n;
        }
        if (!a.join_here) pdl_launch_dependents();   // (the kernel that joins the parts: its wait has no limit)
        if (issuer) umma_commit<false>(bar(C::B_DONE));
        __syncwarp();
        mbar_wait_bounded(bar(C::B_DONE), 0);
    } else if (warp == 17) {
        // ---- copies ----
        const int box_keys = C::CODES ? min((int)C::RAW_KEYS, 1 << shift) : min(BN, 1 << shift), box_shift = 31 - __clz(box_keys), boxes = BN >> box_shift;
        const uint64_t pol = l2_policy_evict_normal();
        int kt = 0, raw = 0;
        while (next_segment()) {
            const TileRange tr = sg.tiles(w);
            const int p0 = sg.p0(w), p1 = sg.p1(w), lo0 = window_begin(p0 < 0 ? 0 : p0, w.window), kv_head = sg.vhead / parts, n = sg.count;
            auto key_of = [&](int j) { return p1 < 0 ? 0 : tr.tile_at(sg.first + j) * BN; };
            // the page of box `lane` of tile j: -1 where no row sees any of it, -2 where the table is wrong
            auto page_of = [&](int j) {
                if (j >= n || lane >= boxes) return -1;
                const int key = key_of(j) + lane * box_keys;
                if (key > p1 || (key + box_keys <= lo0 && key >= w.sinks)) return -1;
                const int page = a.s.page_table[(int64_t)sg.seq * a.s.table_stride + (key >> shift)];
                return page_ok(page, a.c.num_pages) ? page : -2;
            };
            auto cells = [&](int j, int page) { return cell_row(page, kv_head, (key_of(j) + lane * box_keys) & ((1 << shift) - 1), a.c.kv_heads, shift); };
            // 16-key granules of a tile that are copied
            auto granules = [&](unsigned here) {
                unsigned m = 0;
                for (int b = 0; b < boxes; ++b) m |= (here >> b & 1u) ? ((1u << (box_keys / 16)) - 1u) << (b * (box_keys / 16)) : 0u;
                return m;
            };
            auto copy = [&](int j, int page, bool value) {
                if (page == -2) a.status[STATUS_BAD_TABLE] = 1;
                const bool in = page >= 0;
                const unsigned here = __ballot_sync(0xffffffffu, in);
                const int64_t row = in ? cells(j, page) : 0;
                const int tile = kt + j;
                if (!value && lane == 0) *reinterpret_cast<volatile unsigned*>(smem + C::O_HERE + (tile % C::HERE) * 4) = granules(here);
                if (!C::CODES) {
                    const int slot = tile % C::RING, full = (value ? C::B_VFULL : C::B_KFULL) + slot;
                    wait((value ? C::B_VEMPTY : C::B_KEMPTY) + slot, ((tile / C::RING) & 1) ^ 1);
                    if (given_up()) return;
                    const uint32_t dst = base + (value ? C::O_V : C::O_K) + slot * C::TILE;
                    // values that no row sees must not be NaN: their weights are 0.  Such a tile is put right here before it is handed on.
                    const int k0 = key_of(j);
                    const bool fix = value && (k0 + BN - 1 > p1 || (k0 < lo0 && k0 + BN > w.sinks) || granules(here) != 0xFFu);
                    const uint32_t to = bar(fix ? C::B_FIX : full);
                    if (lane == 0) mbar_arrive_expect_tx(to, (uint32_t)(__popc(here) * box_keys * D * 2));
                    __syncwarp();
                    if (in) {
#pragma unroll
                        for (int h = 0; h < C::HALVES; ++h)
                            tma_load_2d(dst + h * (BN * 128) + lane * box_keys * 128, value ? &maps.v_tile : &maps.k_tile, h * 64, (int)row, to, pol);
                    }
                    if (fix) {
                        wait(C::B_FIX, raw & 1);
                        ++raw;
                        const unsigned m = granules(here);
                        for (int x = lane; x < BN * (D / 8); x += 32) {
                            const int rr = x / (D / 8), key = k0 + rr;
                            if (key > p1 || (key < lo0 && key >= w.sinks) || !(m >> (rr >> 4) & 1u)) st_shared16(operand_at(dst, rr, x % (D / 8)), make_uint4(0, 0, 0, 0));
                        }
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar(full));
                    }
                    if (!value && lane == 0) mbar_arrive(bar(C::B_META + tile % C::META));
                } else {
                    // A lane for each box, in the part of the tile that it lies in.
                    const int part = lane * box_keys / C::RAW_KEYS, per = C::RAW_KEYS / box_keys, at = lane * box_keys % C::RAW_KEYS, st = (raw + part) % RAWS;
                    const bool leads = lane < boxes && at == 0;
                    const uint32_t full = bar(C::B_RFULL + st), dst = base + C::O_RAW + st * C::RAW_STAGE;
                    const bool late = leads && !mbar_wait_bounded(bar(C::B_REMPTY + st), (((raw + part) / RAWS) & 1) ^ 1);
                    if (__any_sync(0xffffffffu, late)) {
                        *dead = 1;
                        *a.status = 32;
                    }
                    if (given_up()) return;
                    __syncwarp();   // (what lane 0 has noted is read behind any of these barriers)
                    if (leads) mbar_arrive_expect_tx(full, (uint32_t)(__popc(here >> lane & ((1u << per) - 1u)) * box_keys * (D + (value ? 0 : 4))));
                    __syncwarp();
                    if (in) {
                        bulk_g2s(dst + at * D, (const uint8_t*)(value ? a.c.v : a.c.k) + row * D, box_keys * D, full, pol);
                        if (!value) {
                            bulk_g2s(dst + C::RAW + at * 2, a.c.k_scale + row, box_keys * 2, full, pol);
                            bulk_g2s(dst + C::RAW + 2 * C::RAW_KEYS + at * 2, a.c.v_scale + row, box_keys * 2, full, pol);
                        }
                    }
                    raw += BN / C::RAW_KEYS;
                }
            };
            // in the order in which they are used: K 0, K 1, then V j and K j + 2
            int pages[3] = {page_of(0), page_of(1), page_of(2)};
            copy(0, pages[0], false);
            if (n > 1) copy(1, pages[1], false);
            for (int j = 0; j < n; ++j) {
                const int next = page_of(j + 3);
                // Cells of 128 dims leave room for four parts in flight, too few for the memory's latency: what comes next waits in the L2 (32 x 24 tokens to
                // 8192 positions, 16 heads to 4: e4m3 180 -> 145 us, int8 186 -> 177).  With 64 dims there are twelve (93 -> 103 us with this).
                if (C::CODES && D == 128 && next >= 0) {
                    const int64_t row = cells(j + 3, next);
                    bulk_prefetch_l2((const uint8_t*)a.c.k + row * D, box_keys * D);
                    bulk_prefetch_l2((const uint8_t*)a.c.v + row * D, box_keys * D);
                }
                copy(j, pages[0], true);
                if (j + 2 < n) copy(j + 2, pages[2], false);
                pages[0] = pages[1];
                pages[1] = pages[2];
                pages[2] = next;
            }
            kt += n;
        }
        if (given_up()) {   // what was asked for must land before the block's memory is given back
            if (C::CODES)
                for (int i = raw < RAWS ? 0 : raw - RAWS; i < raw; ++i) mbar_wait_bounded(bar(C::B_RFULL + i % RAWS), (i / RAWS) & 1);
            else
                for (const long long t0 = clock64(); clock64() - t0 < WAIT_CYCLES;) {}   // (copies that a broken order left on either ring: time enough for any)
        }
    } else if (C::CODES && warp >= C::FIRST_EXPANDER) {
        // ---- codes to operands ----
        // Each warp has every other part of a tile.  A thread takes the same 16 codes of every ROWS-th key: its place in a row of operands, and so the
        // swizzle, stays.
        constexpr int ROWS = 32 / (D / 16), PIECES = C::RAW_KEYS / ROWS, PERIOD = 8 / ROWS;   // (the swizzle comes round after 8 rows)
        const int row0 = lane / (D / 16), piece = lane % (D / 16);
        const bool swap = D == 128 && (piece & 4);   // (the two columns of 64 dims share banks: neighbours take opposite pieces first)
        uint32_t off0[PERIOD], off1[PERIOD];
#pragma unroll
        for (int y = 0; y < PERIOD; ++y) {
            off0[y] = operand_at(0, row0 + y * ROWS, 2 * piece + (swap ? 1 : 0));
            off1[y] = operand_at(0, row0 + y * ROWS, 2 * piece + (swap ? 0 : 1));
        }
        int kt = 0, raw = 0;
        while (next_segment()) {
            const TileRange tr = sg.tiles(w);
            const int p0 = sg.p0(w), p1 = sg.p1(w), lo0 = window_begin(p0 < 0 ? 0 : p0, w.window), n = sg.count;
            auto expand = [&](int j, bool value) {
                const int tile = kt + j, slot = tile % C::RING, mt = tile % C::META;
                const int k0 = p1 < 0 ? 0 : tr.tile_at(sg.first + j) * BN;
                wait((value ? C::B_VEMPTY : C::B_KEMPTY) + slot, ((tile / C::RING) & 1) ^ 1);
                const uint32_t dst = base + (value ? C::O_V : C::O_K) + slot * C::TILE;
                for (int part = warp - C::FIRST_EXPANDER; part < BN / C::RAW_KEYS; part += C::EXPANDERS) {
                    const int st = (raw + part) % RAWS;
                    wait(C::B_RFULL + st, ((raw + part) / RAWS) & 1);
                    const uint8_t* src = smem + C::O_RAW + st * C::RAW_STAGE;
                    const unsigned here = *reinterpret_cast<volatile unsigned*>(smem + C::O_HERE + tile % C::HERE * 4);
                    const bool fix = value && (k0 + BN - 1 > p1 || (k0 < lo0 && k0 + BN > w.sinks) || here != 0xFFu);
                    float ks = 0.f, vs = 0.f;
                    if (!value) {
                        ks = half_float(reinterpret_cast<const uint16_t*>(src + C::RAW)[lane]);
                        vs = half_float(reinterpret_cast<const uint16_t*>(src + C::RAW + 2 * C::RAW_KEYS)[lane]);
                    }
                    auto pieces = [&](auto fixed) {
#pragma unroll
                        for (int b = 0; b < PIECES; b += 4) {
                            uint4 q[4];
#pragma unroll
                            for (int y = 0; y < 4; ++y) q[y] = reinterpret_cast<const uint4*>(src)[lane + (b + y) * 32];
                            if (b + 4 == PIECES) {   // all of the part has been read: the next one may come (given back at the end: int8, 128 dims, 641 us instead of 598)
                                __syncwarp();
                                if (lane == 0) mbar_arrive(bar(C::B_REMPTY + st));
                            }
#pragma unroll
                            for (int y = 0; y < 4; ++y) {
                                // values that no row sees must not be NaN: their weights are 0
                                const int rr = part * C::RAW_KEYS + row0 + (b + y) * ROWS, key = k0 + rr;
                                if (decltype(fixed)::value && (key > p1 || (key < lo0 && key >= w.sinks) || !(here >> (rr >> 4) & 1u))) q[y] = make_uint4(0, 0, 0, 0);
                                uint4 lo, hi;
                                codes_to_half2x2<FMT>(q[y].x, lo.x, lo.y);
                                codes_to_half2x2<FMT>(q[y].y, lo.z, lo.w);
                                codes_to_half2x2<FMT>(q[y].z, hi.x, hi.y);
                                codes_to_half2x2<FMT>(q[y].w, hi.z, hi.w);
                                const uint32_t to = dst + part * (C::RAW_KEYS * 128) + (b + y) / PERIOD * (8 * 128);
                                st_shared16(to + off0[(b + y) % PERIOD], swap ? hi : lo);
                                st_shared16(to + off1[(b + y) % PERIOD], swap ? lo : hi);
                            }
                        }
                    };
                    if (fix) pieces(std::true_type());
                    else pieces(std::false_type());
                    if (!value) {
                        const int key = part * C::RAW_KEYS + lane;
                        // (the scales of keys that no row sees may be anything)
                        const bool seen = k0 + key <= p1 && (k0 + key >= lo0 || k0 + key < w.sinks) && (here >> (key >> 4) & 1u);
                        const float b = seen ? fmaf(ks, 0.f, lg2(vs)) : 0.f;   // (an infinite scale as a NaN: the formula knows what codes of 0 make of it)
                        float* meta = reinterpret_cast<float*>(smem + C::O_META + mt * C::META_BYTES) + key;
                        meta[0] = seen ? ks * scale2 : 1.f;
                        meta[BN] = b;
                        meta[2 * BN] = ex2(-b);
                    }
                }
                raw += BN / C::RAW_KEYS;
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar((value ? C::B_VFULL : C::B_KFULL) + slot));
                    if (!value) mbar_arrive(bar(C::B_META + mt));
                }
            };
            expand(0, false);
            if (n > 1) expand(1, false);
            for (int j = 0; j < n; ++j) {
                expand(j, true);
                if (j + 2 < n) expand(j + 2, false);
            }
            kt += n;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 16) tmem_dealloc<false>(tmem, 512);
}

// Joins the parts of items that blocks share: block (b, y) the rows 32 y .. of the item that block b of the kernel above began and did not finish.
constexpr int JOIN_THREADS = 256;
template <int FMT, int D, bool TREE>
__global__ void __launch_bounds__(JOIN_THREADS) attention_join_kernel(const AttnArgs a) {
    pdl_wait_prior_grid();
    const int b0 = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int4 it = a.items[b0];
    if (it.x < 0) return;
    WorkShape w;
    const int parts = (a.group + 127) / 128;
    w.group = (a.group + parts - 1) / parts;
    w.tokens = 2 * (128 / w.group);
    w.tree_words = TREE ? a.tree_words : 0;
    const SeqWork q = load_seq(a.s, w, it.x);
    const int t0 = it.z * w.tokens, t1 = min(t0 + w.tokens, q.n) - 1, per = w.tokens / 2, r = blockIdx.y * 32 + lane, i = r >> 7;
    const int t = t0 + i * per + (r & 127) / w.group, hg = (it.y % parts) * w.group + (r & 127) % w.group;
    const bool on = (r & 127) < per * w.group && t <= min(t1, t0 + (i + 1) * per - 1) && hg < a.group;
    if (!__syncthreads_or(on)) return;
    const int row = q.row0 + t, head = it.y / parts * a.group + hg, pos = q.len - q.n + (TREE ? 0 : t);
    const float4* base = reinterpret_cast<const float4*>(a.parts);
    auto part = [&](int b) { return base + (int64_t)(2 * b + (b == b0 ? 1 : 0)) * (ATTN_CHUNK_PART / 16); };
    float m = -INFINITY;
    for (int b = b0; b <= it.w; ++b) m = fmaxf(m, reinterpret_cast<const float2*>(part(b) + 64 * D)[r].x);
    constexpr int N = D / 32;   // quads of dims of a warp
    float4 o[N] = {};
    float l = 0.f;
#pragma unroll 2
    for (int b = b0; b <= it.w; ++b) {
        const float4* p = part(b);
        const float2 s = reinterpret_cast<const float2*>(p + 64 * D)[r];
        float4 v[N];
#pragma unroll
        for (int x = 0; x < N; ++x) v[x] = p[(warp * N + x) * 256 + r];
        const float f = s.x == -INFINITY ? 0.f : exp2f(s.x - m);
        l += s.y * f;
#pragma unroll
        for (int x = 0; x < N; ++x) {
            o[x].x += v[x].x * f;
            o[x].y += v[x].y * f;
            o[x].z += v[x].z * f;
            o[x].w += v[x].w * f;
        }
    }
    const float inv = 1.f / l;
    bool fine = l > 0.f && l < INFINITY;
#pragma unroll
    for (int x = 0; x < N; ++x) {
        o[x].x *= inv;
        o[x].y *= inv;
        o[x].z *= inv;
        o[x].w *= inv;
        fine = fine && fabsf(o[x].x) < HALF_END && fabsf(o[x].y) < HALF_END && fabsf(o[x].z) < HALF_END && fabsf(o[x].w) < HALF_END;
    }
    __shared__ unsigned bad[JOIN_THREADS / 32];
    const unsigned mine = __ballot_sync(0xffffffffu, on && !fine);
    if (lane == 0) bad[warp] = mine;
    __syncthreads();
    unsigned again = 0;
#pragma unroll
    for (int x = 0; x < JOIN_THREADS / 32; ++x) again |= bad[x];
    if (on && !(again >> lane & 1u)) {
        uint2* out = reinterpret_cast<uint2*>(a.out + (int64_t)row * a.o_stride + (int64_t)head * D) + warp * N;
#pragma unroll
        for (int x = 0; x < N; ++x) out[x] = make_uint2(floats_half2(o[x].x, o[x].y), floats_half2(o[x].z, o[x].w));
    }
    if (!again) pdl_launch_dependents();   // (the rest may take long)
    int k = 0;   // rows that are not finite, or see nothing: from the formula once more, a warp each
    for (unsigned left = again; left; left &= left - 1, ++k) {
        const int from = __ffs(left) - 1;
        const int r2 = __shfl_sync(0xffffffffu, row, from), h2 = __shfl_sync(0xffffffffu, head, from), p2 = __shfl_sync(0xffffffffu, pos, from);
        if (k % (JOIN_THREADS / 32) == warp && !attend_row<FMT, D, TREE>(a, it.x, q.len, p2, r2, h2) && lane == 0) a.status[STATUS_BAD_TABLE] = 1;
    }
}

template <int FMT, int D, bool TREE>
cudaError_t launch_one(const AttnArgs& a, const AttnMaps& maps, int blocks, cudaStream_t st, bool pdl, int* kernels) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(Chunk<FMT, D>::THREADS);
    cfg.dynamicSmemBytes = Chunk<FMT, D>::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, attention_chunk_kernel<FMT, D, TREE>, maps, a);
    *kernels = a.join_here ? 1 : 2;
    if (e != cudaSuccess || a.join_here) return e;
    cfg.gridDim = dim3((unsigned)blocks, 8);
    cfg.blockDim = dim3(JOIN_THREADS);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, attention_join_kernel<FMT, D, TREE>, a);
}
template <int FMT, int D>
cudaError_t launch(const AttnArgs& a, const AttnMaps& maps, int blocks, cudaStream_t st, bool pdl, int* kernels) {
    return a.tree ? launch_one<FMT, D, true>(a, maps, blocks, st, pdl, kernels) : launch_one<FMT, D, false>(a, maps, blocks, st, pdl, kernels);
}

template <int FMT, int D>
cudaError_t configure() {
    const cudaError_t e = cudaFuncSetAttribute(attention_chunk_kernel<FMT, D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Chunk<FMT, D>::SMEM);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(attention_chunk_kernel<FMT, D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Chunk<FMT, D>::SMEM);
}

}  // namespace

cudaError_t attention_chunk_configure() {
    cudaError_t e;
    if ((e = configure<KV_FP16, 64>()) != cudaSuccess || (e = configure<KV_FP16, 128>()) != cudaSuccess || (e = configure<KV_INT8, 64>()) != cudaSuccess ||
        (e = configure<KV_INT8, 128>()) != cudaSuccess || (e = configure<KV_FP8, 64>()) != cudaSuccess)
        return e;
    return configure<KV_FP8, 128>();
}

// An item's parts are joined by the last block to have one, or, where there are several to an item, by a kernel of their own, in more blocks.
// Here / apart, us: 2 x 4096 tokens under a window of 1024 (16 heads to 8 of 64 dims, fp16; items cut in 1 to 2 parts) 98.5 / 100.8; 16 x 64 tokens to 2048
// (32 heads to 8 of 128 dims, e4m3; 1 to 2) 78.0 / 80.3; 8 x 20 to 4096 (28 to 4 of 128, fp16; 5) 34.9 / 33.1; 1 x 17 to 4096 (32 to 4 of 64; 32) 23.5 / 18.1;
// 1 x 32 to 32768 (8 to 1 of 128; 148) 212 / 62.
constexpr int PARTS_HERE = 2;

cudaError_t launch_attention_chunk(const AttnArgs& given, const AttnMaps& maps, int sm_count, cudaStream_t st, bool pdl, int* kernels) {
    const int blocks = sm_count < ATTN_MAX_BLOCKS ? sm_count : ATTN_MAX_BLOCKS;
    AttnArgs a = given;
    const int parts = (a.group + 127) / 128, tokens = 2 * (128 / ((a.group + parts - 1) / parts)), tiles = (a.s.num_rows - 1) / tokens + 1;
    a.join_here = (long long)a.c.kv_heads * parts * (a.s.num_seqs > tiles ? a.s.num_seqs : tiles) * PARTS_HERE >= blocks;
    if (a.c.fmt == KV_FP16) return a.c.dim == 64 ? launch<KV_FP16, 64>(a, maps, blocks, st, pdl, kernels) : launch<KV_FP16, 128>(a, maps, blocks, st, pdl, kernels);
    if (a.c.fmt == KV_INT8) return a.c.dim == 64 ? launch<KV_INT8, 64>(a, maps, blocks, st, pdl, kernels) : launch<KV_INT8, 128>(a, maps, blocks, st, pdl, kernels);
    return a.c.dim == 64 ? launch<KV_FP8, 64>(a, maps, blocks, st, pdl, kernels) : launch<KV_FP8, 128>(a, maps, blocks, st, pdl, kernels);
}

}  // namespace nnb
