// Beam search's selection: the best continuations of each group of beams.
//
//   total(b, v) = score_b + ((x_bv - m_b) - log sum_w exp(x_bw - m_b))      x fp16 logits, m_b the row's maximum
//
// and of an ended beam only (b, eos) with score_b.  The largest totals come first, of equal ones the lowest beam, then the lowest token.
//
// Bound by the logits' bytes, each read once.  A row is cut into segments, a block each; a thread has every 256th vector of 8 values of its segment, its share, and
// keeps their maximum and the sum of exponentials behind it.  The row's best `picks` values lie in those shares whose maxima are the `picks`
// best ones: every other share has `picks` values before all of its own.  So no value needs a place in a list while the logits stream by, whatever
// their order.  The row's last block finds those shares, reads them again, a value to a thread, and has the row's candidates; the group's last
// block joins its rows' lists.  Where there are few blocks each does so for its segment, and the group's last one joins the segments' lists (DIRECT).
// Within a row the fp16 values and the tokens decide, exactly.  Across rows the totals do, in 64 bits.  Exponentials are taken of differences to the largest value that their warp has seen, in 32 bits.
// A maximum is exactly 1; a value d below it is off by what rounding takes from d and from its product with log2 e (half a step each), by that constant (d 2^-26) and by
// ex2 (2^-22, measured: 0.61 of that), equal values by the same.  From there on sums are scaled in 64 bits (a maximum that rises, warps, segments): in 32 bits and for each thread, 64 rising maxima
// of a thread put the logarithm 2 2^-20 off.  So a warp's 65536 values, one peak and the others equal, 6 to 8 below it, are the worst: 1.5 2^-20, with five steps of adding up, whatever the row's length, and
// totals that are 2^-18 apart come in order.  (Measured of such rows: 0.9 2^-20 between two; of 151936 values of N(0, 2.5), whose errors are different ones, some 2^-27 each.)  For that the
// serving batch below takes 3 % longer.  Everything depends on differences alone: rows that are shifted against each other give the same logarithms.
// 64 groups of 8 beams of 151936 fp16 logits, 16 picks: 46 us (3.4 TB/s; the bytes alone 24).  The exponential unit has 36 thousand clocks of it, the logits altogether some 54 (28 us),
// the last rows' steps behind them 8 us.  One group of 4 beams of 49152: 8.5 us, all of it such steps.
#include <cuda_fp16.h>

#include "kv_branch.h"
#include "ptx.cuh"

namespace nnb {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32, BATCH = 4;
constexpr int TOPS = MOST_PICKS / 4;        // maxima of a warp that are compared with the other warps'
constexpr int ROOM = 3136;                  // keys that a block compares with one another
constexpr int DIRECT_MOST = 1024, DIRECT_LISTS = 128;   // candidates and segments of a group that its last block joins without the rows' lists
constexpr unsigned NO_VALUE = 0x03FFu;      // the code of -infinity

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// the largest number of a warp (NaN: of the others)
__device__ __forceinline__ float warp_max(float x) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}
// fp16 numbers in order as whole ones, both zeros the same
__device__ __forceinline__ unsigned code_of(uint16_t h) {
    if (h == 0x8000u) h = 0;
    return h & 0x8000u ? 0xFFFFu & ~(unsigned)h : h | 0x8000u;
}
__device__ __forceinline__ float value_of(unsigned code) {
    return __half2float(__ushort_as_half((uint16_t)(code & 0x8000u ? code & 0x7FFFu : ~code)));
}

// What follows is short code: a block goes through the kernel once, and instructions that no block of its SM has used before come from the L2 (unrolled,
// with sorting networks: joining the lists of 4 beams took 33 thousand clocks, of which two thousand were work).

// The places among `n` different keys of all of them, by the whole block: take(place, key).  Few keys have several threads each, next to one another, which go through a
// part of the list.
using Key = unsigned long long;
template <class Take>
__device__ __forceinline__ void places_of(const Key* keys, int n, Take&& take) {
    const int shift = n <= THREADS / 8 ? 3 : n <= THREADS / 4 ? 2 : n <= THREADS / 2 ? 1 : 0, parts = 1 << shift, part = threadIdx.x & (parts - 1);
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += THREADS >> shift) {
        const int i = i0 + (threadIdx.x >> shift);
        const Key mine = i < n ? keys[i] : ~0ull;
        int larger = 0, also = 0;
#pragma unroll 4
        for (int p = part; p < n / 2; p += parts) {
            const ulonglong2 two = reinterpret_cast<const ulonglong2*>(keys)[p];
            larger += two.x > mine;
            also += two.y > mine;
        }
        if ((n & 1) && part == 0) larger += keys[n - 1] > mine;
        larger += also;
#pragma unroll 1
        for (int d = 1; d < parts; d <<= 1) larger += __shfl_xor_sync(0xffffffffu, larger, d);
        if (i < n && part == 0) take(larger, mine);
    }
}

constexpr double LN2 = 0.693147180559945309417;
// exp(x), x <= 0: 2^n times the exponential's series of what is left, at most ln 2 / 2 (11 terms: 2^-41)
__device__ __forceinline__ double exp_of(double x) {
    if (!(x > -700.)) return x == x ? 0. : x;
    const double n = rint(x * (1. / LN2)), f = fma(n, -LN2, x);
    double p = 1. / 3628800.;
    p = fma(p, f, 1. / 362880.);
    p = fma(p, f, 1. / 40320.);
    p = fma(p, f, 1. / 5040.);
    p = fma(p, f, 1. / 720.);
    p = fma(p, f, 1. / 120.);
    p = fma(p, f, 1. / 24.);
    p = fma(p, f, 1. / 6.);
    p = fma(p, f, 0.5);
    p = fma(p, f, 1.);
    p = fma(p, f, 1.);
    return p * __longlong_as_double((long long)(n + 1023.) << 52);
}
// log(x), x positive and finite: with x = 2^n m and z = (m - 1) / (m + 1), n ln 2 + 2 (z + z^3 / 3 + z^5 / 5 + ..); |z| <= 0.172 (9 terms: 2^-50)
__device__ __forceinline__ double log_of(double x) {
    const long long bits = __double_as_longlong(x);
    int n = (int)(bits >> 52) - 1023;
    double m = __longlong_as_double((bits & 0xFFFFFFFFFFFFFll) | 1023ll << 52);
    if (m > 1.4142135623730951) {
        m *= 0.5;
        ++n;
    }
    const double d = m + 1.;
    double r = (double)__fdividef(1.f, (float)d);   // its reciprocal, by Newton's method
    r = r * fma(-d, r, 2.);
    r = r * fma(-d, r, 2.);
    const double z = (m - 1.) * r, q = z * z;
    double p = 1. / 17.;
    p = fma(p, q, 1. / 15.);
    p = fma(p, q, 1. / 13.);
    p = fma(p, q, 1. / 11.);
    p = fma(p, q, 1. / 9.);
    p = fma(p, q, 1. / 7.);
    p = fma(p, q, 1. / 5.);
    p = fma(p, q, 1. / 3.);
    p = fma(p, q, 1.);
    return fma((double)n, LN2, 2. * z * p);
}

// A row of logits as vectors of 8 tokens, wherever the row begins (so that equal rows are added up in the same order and give the same bits).
// Behind the row's end there is -infinity.
struct Row {
    const uint16_t* p;
    int vocab;
    __device__ __forceinline__ Row(const uint16_t* row, int v) : p(row), vocab(v) {}
    __device__ __forceinline__ int vectors() const { return (vocab + 7) / 8; }
    // Of these vectors, whole ones at 16-byte boundaries, the first `plain` are.
    __device__ __forceinline__ int plain() const { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 ? vocab / 8 : 0; }
    __device__ __forceinline__ uint4 load_plain(int i) const {
        uint4 x;
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(p + (int64_t)8 * i));
        return x;
    }
    __device__ __forceinline__ uint4 load(int i) const { return i < plain() ? load_plain(i) : load_any(p, vocab, i); }
    static __device__ __noinline__ uint4 load_any(const uint16_t* p, int vocab, int i) {
        const int off = (int)(reinterpret_cast<uintptr_t>(p) & 15);   // the same for all of the row's vectors
        const uint16_t* const at = p + (int64_t)8 * i;
        uint32_t w[8];
        if (off != 0 && i > 0 && 8 * i + 16 - off / 2 <= vocab) {   // two pieces at 16-byte boundaries; the second is the next thread's first
            const uint4* const two = reinterpret_cast<const uint4*>(at - off / 2);
            const uint4 a = __ldg(two), b = __ldg(two + 1);
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
            if (off & 8) {
#pragma unroll
                for (int j = 0; j < 6; ++j) w[j] = w[j + 2];
            }
            if (off & 4) {
#pragma unroll
                for (int j = 0; j < 5; ++j) w[j] = w[j + 1];
            }
            if (off & 2) {
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], 16);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = 8 * i + 2 * j;
                w[j] = (t < vocab ? at[2 * j] : 0xFC00u) | (uint32_t)(t + 1 < vocab ? at[2 * j + 1] : 0xFC00u) << 16;
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
__device__ __forceinline__ __half2 as_half2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
__device__ __forceinline__ __half2 most_of(const uint4& x) { return __hmax2(__hmax2(as_half2(x.x), as_half2(x.y)), __hmax2(as_half2(x.z), as_half2(x.w))); }
__device__ __forceinline__ __half most_of(__half2 x) { return __hmax(__low2half(x), __high2half(x)); }

struct Part {   // of a segment
    unsigned key[THREADS];   // of each thread's share: code of its largest value << 16 | 0xFFFF - the vector of the segment where that is first
    double sum;              // of exponentials behind the segment's largest value
    unsigned top, unused;    // that value's code
};
struct Candidates {   // of a row, the best first
    Key total[MOST_PICKS];   // order_of, the last five bits replaced by 31 - beam: of equal totals the lowest beam is first; 0: none
    int token[MOST_PICKS];
};
struct Best {   // of a segment, the best first
    Key key[MOST_PICKS];   // value's code << 32 | 0xFFFFFFFF - token; 0: none
    double sum;            // as in Part
    unsigned top, unused[29];
};
static_assert(sizeof(Part) == BEAM_PART_BYTES && sizeof(Candidates) == BEAM_ROW_BYTES && sizeof(Best) == BEAM_ROW_BYTES, "workspace");
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t d, x = *reinterpret_cast<const uint64_t*>(&a), y = *reinterpret_cast<const uint64_t*>(&b);
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(x), "l"(y));
    return *reinterpret_cast<const float2*>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t d, x = *reinterpret_cast<const uint64_t*>(&a), y = *reinterpret_cast<const uint64_t*>(&b);
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(x), "l"(y));
    return *reinterpret_cast<const float2*>(&d);
}

constexpr float LOG2E = 1.4426950408889634f;

// 64-bit numbers in order as whole ones, none of them 0; and back
__device__ __forceinline__ unsigned long long order_of(double t) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(t == 0 ? 0. : t);
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double total_of(unsigned long long u) { return __longlong_as_double((long long)(u >> 63 ? u & ~(1ull << 63) : ~u)); }

// Whether this block is the last of `n` to arrive; what all of their threads have written before is visible to it then.  There is no barrier behind the reads of
// the flag: between two of these calls nobody else writes it, and the next one begins with a barrier.
__device__ __forceinline__ bool last_of(unsigned* counter, unsigned n, volatile int* flag) {
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned before;
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
        if (before == n - 1) *counter = 0u;
        *flag = before == n - 1;
    }
    __syncthreads();
    return *flag != 0;
}

// The group's picks from its segments' candidates: rows' sums, totals, and of those that may be among the picks the place of each.
struct JoinRoom {
    ulonglong2 left[DIRECT_MOST];   // total as in Candidates, and key as in Best
    Key some[DIRECT_LISTS];
    double norm[MOST_BEAMS], most[MOST_BEAMS];
    unsigned bar;                   // of totals' upper halves
    int count, there;
};
__device__ __forceinline__ void join_segments(const BeamSelectArgs& a, int group, JoinRoom& room) {
    const int tid = threadIdx.x, lane = tid & 31, picks = a.picks, per_beam = a.segs * picks, num = a.beams * a.segs, n = num * picks;
    const Best* const lists = reinterpret_cast<const Best*>(a.rows) + (int64_t)group * num;
    constexpr int EACH = DIRECT_MOST / THREADS;
    Key key[EACH], total[EACH];
    float score[EACH];
    bool ended[EACH];
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
        key[u] = total[u] = 0;
        score[u] = 0.f;
        ended[u] = false;
        const int i = tid + u * THREADS;
        if (i < n) {
            const int l = i / picks, b = i / per_beam;
            key[u] = __ldcg(&lists[l].key[i - l * picks]);   // (of rows that are not looked at: left from another call)
            score[u] = a.score[group * a.beams + b];
            ended[u] = a.done && a.done[group * a.beams + b] != 0;
        }
    }
#pragma unroll 1
    for (int b = tid >> 5; b < a.beams; b += WARPS) {   // a row to a warp
        const Best* const p = lists + b * a.segs;
        const unsigned top0 = lane < a.segs ? __ldcg(&p[lane].top) : 0u;
        const double y0 = lane < a.segs ? __ldcg(&p[lane].sum) : 0.;
        unsigned top = top0;
        for (int s = lane + 32; s < a.segs; s += 32) top = max(top, __ldcg(&p[s].top));
        top = __reduce_max_sync(0xffffffffu, top);
        const double most = value_of(top);
        double sum = y0 != 0 ? top0 > NO_VALUE ? y0 * exp_of((double)value_of(top0) - most) : y0 : 0.;
        for (int s = lane + 32; s < a.segs; s += 32) {
            const unsigned c = __ldcg(&p[s].top);
            const double y = __ldcg(&p[s].sum);
            if (y != 0) sum += c > NO_VALUE ? y * exp_of((double)value_of(c) - most) : y;
        }
#pragma unroll 1
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) {
            room.norm[b] = sum > 0 && sum < INFINITY && most < INFINITY ? log_of(sum) : -1.;   // (-1: a NaN or an infinity among the values, no candidates)
            room.most[b] = most;
        }
    }
    const bool few = n <= THREADS / 4;   // (all are compared with all)
    if (tid == 0) {
        room.bar = few ? 0u : ~0u;
        room.count = room.there = 0;
    }
    __syncthreads();
    // Where `each`-th totals of that many lists are not below a total, it is not below the last pick's.
    const int each = (picks + num - 1) / num, enough = (picks + each - 1) / each;
    int there = 0;
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
        const int i = tid + u * THREADS;
        if (i < n) {
            const int l = i / picks, b = i / per_beam;
            if (ended[u]) key[u] = i == b * per_beam ? 0xFFFFFFFFu - (unsigned)a.eos : 0u;
            if (key[u] != 0 && fabsf(score[u]) < INFINITY && (ended[u] || room.norm[b] >= 0)) {
                const double t = ended[u] ? (double)score[u] : (double)score[u] + (((double)value_of((unsigned)(key[u] >> 32)) - room.most[b]) - room.norm[b]);
                total[u] = (order_of(t) & ~31ull) | (unsigned)(31 - b);
                ++there;
            }
            if (i - l * picks == each - 1) room.some[l] = total[u];
        }
    }
    there = __reduce_add_sync(0xffffffffu, there);
    if (lane == 0 && there) atomicAdd(&room.there, there);
    if (!few) {
        __syncthreads();
        places_of(room.some, num, [&](int place, Key k) {
            if (place < enough) atomicMin(&room.bar, (unsigned)(k >> 32));   // (0: fewer lists have so many)
        });
    }
    __syncthreads();   // (scores and flags have been read: they may be the outputs)
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
        if (u * THREADS >= n) break;
        const bool stays = total[u] != 0 && (unsigned)(total[u] >> 32) >= room.bar;
        const unsigned who = __ballot_sync(0xffffffffu, stays);
        int to = 0;
        if (lane == 0 && who) to = atomicAdd(&room.count, __popc(who));
        to = __shfl_sync(0xffffffffu, to, 0) + __popc(who & ((1u << lane) - 1u));
        if (stays) room.left[to] = make_ulonglong2(total[u], key[u]);
    }
    __syncthreads();
    const int left = room.count, shift = left <= THREADS / 8 ? 3 : left <= THREADS / 4 ? 2 : left <= THREADS / 2 ? 1 : 0, threads = 1 << shift, part = tid & (threads - 1);
#pragma unroll 1
    for (int i0 = 0; i0 < left; i0 += THREADS >> shift) {
        const int i = i0 + (tid >> shift);
        const ulonglong2 mine = room.left[i < left ? i : 0];
        int place = 0;
#pragma unroll 2
        for (int j = part; j < left; j += threads) {
            const ulonglong2 other = room.left[j];
            place += other.x > mine.x || (other.x == mine.x && other.y > mine.y);
        }
#pragma unroll 1
        for (int d = 1; d < threads; d <<= 1) place += __shfl_xor_sync(0xffffffffu, place, d);
        if (i < left && part == 0 && place < picks) {
            const int64_t o = (int64_t)group * picks + place;
            const int token = (int)(0xFFFFFFFFu - (unsigned)mine.y);
            a.out_score[o] = (float)total_of(mine.x);
            a.out_token[o] = token;
            a.out_parent[o] = 31 - (int)(mine.x & 31);
            if (a.out_done) a.out_done[o] = token == a.eos;
        }
    }
    if (tid >= room.there && tid < picks) {   // no more candidates
        const int64_t o = (int64_t)group * picks + tid;
        a.out_score[o] = -INFINITY;
        a.out_token[o] = a.out_parent[o] = -1;
        if (a.out_done) a.out_done[o] = 0;
    }
}

// (six blocks to an SM, for loads in flight: with five and more registers 47.4 us where it is 45.8)
template <bool DIRECT>
__global__ void __launch_bounds__(THREADS, DIRECT ? 4 : 6) beam_select_kernel(const BeamSelectArgs a) {
    __shared__ __align__(16) Key found[ROOM];
    __shared__ Key best[MOST_PICKS];
    __shared__ __align__(16) Key best_of[WARPS * TOPS];
    __shared__ unsigned tops[WARPS];
    __shared__ double sums[WARPS];
    __shared__ int flag, count, homes[MOST_PICKS];
    __shared__ unsigned bar;   // (a word of its own: a warp may still be reading what last_of has left in its flag)
    static_assert(sizeof(Candidates) * MOST_BEAMS <= sizeof(found) && sizeof(JoinRoom) <= sizeof(found), "room");
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x / a.segs, seg = blockIdx.x - row * a.segs, group = row / a.beams, picks = a.picks;
    // A beam that has ended, or has no score, is not looked at.
    const float score = a.score[row];
    const bool scored = fabsf(score) < INFINITY, looked_at = scored && !(a.done && a.done[row] != 0);
    constexpr bool direct = DIRECT;
    unsigned own = 0;          // (direct) this thread's share as in Part::key
    Part* const parts = reinterpret_cast<Part*>(a.parts);
    Best& list = reinterpret_cast<Best*>(a.rows)[blockIdx.x];   // (direct)
    const Row x(a.logits + (int64_t)row * a.stride, a.vocab);
    auto segment_sum = [&](double& sum, unsigned& top) {   // of the warps' ones, by a warp
        const unsigned mine = lane < WARPS ? tops[lane] : 0u, most = __reduce_max_sync(0xffffffffu, mine);
        double s = lane < WARPS ? sums[lane] : 0.0;
        if (s != 0) s *= exp_of((double)value_of(mine) - (double)value_of(most));
#pragma unroll 1
        for (int d = WARPS / 2; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (lane == 0) {
            sum = s;
            top = most;
        }
    };
    if (looked_at) {
        const int begin = seg * a.per_seg, end = min(x.vectors(), begin + a.per_seg), plain = min(x.plain(), end);
        __half most = __ushort_as_half(0xFC00);
        float peak = -INFINITY;        // the warp's largest value: sums are of exponentials of differences to that
        float sum = 0.f, rest = 0.f;   // (rest: what rounding has taken from the sum)
        int at = 0;
#pragma unroll 1
        for (int i0 = begin + tid; i0 - lane < end; i0 += THREADS * BATCH) {   // (whole warps stay together)
            uint4 v[BATCH];
            if (i0 + (BATCH - 1) * THREADS < plain) {
#pragma unroll
                for (int j = 0; j < BATCH; ++j) v[j] = x.load_plain(i0 + j * THREADS);
            } else {
#pragma unroll
                for (int j = 0; j < BATCH; ++j) v[j] = i0 + j * THREADS < end ? x.load(i0 + j * THREADS) : make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u);
            }
            __half2 m[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) m[j] = most_of(v[j]);
            const __half up = most_of(__hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3])));
            const float higher = warp_max(__half2float(up));
            if (higher > peak) {   // (of the whole warp)
                if (peak > -INFINITY) {
                    const double all = ((double)sum + (double)rest) * exp_of((double)peak - (double)higher);
                    sum = (float)all;
                    rest = (float)(all - (double)sum);
                }
                peak = higher;
            }
            if (__hgt(up, most)) {
                most = up;
                int j = 0;
                while (j < BATCH - 1 && !__heq(most_of(j == 0 ? m[0] : j == 1 ? m[1] : m[2]), up)) ++j;
                at = i0 + j * THREADS - begin;
            }
            const float ref = peak == -INFINITY ? 0.f : -peak;
            float2 s[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
                float2 e[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float2 t = mul2(add2(__half22float2(as_half2(w[q])), make_float2(ref, ref)), make_float2(LOG2E, LOG2E));
                    e[q] = make_float2(ex2(t.x), ex2(t.y));
                }
                s[j] = add2(add2(e[0], e[1]), add2(e[2], e[3]));
            }
            const float2 both = add2(add2(s[0], s[1]), add2(s[2], s[3]));
            // the sum's rounding is kept (D. Knuth, The Art of Computer Programming 2, 4.2.2)
            const float more = both.x + both.y, whole = __fadd_rn(sum, more), back = __fsub_rn(whole, sum);
            rest += __fadd_rn(__fsub_rn(sum, __fsub_rn(whole, back)), __fsub_rn(more, back));
            sum = whole;
        }
        Part& part = parts[blockIdx.x];
        const unsigned code = code_of(__half_as_ushort(most));
        own = code > NO_VALUE ? code << 16 | (0xFFFFu - at) : 0u;
        if (!direct) part.key[tid] = own;
        double whole = (double)sum + (double)rest;
#pragma unroll 1
        for (int d = 16; d > 0; d >>= 1) whole += __shfl_xor_sync(0xffffffffu, whole, d);
        if (lane == 0) {
            tops[warp] = code_of(__half_as_ushort(__float2half_rn(peak)));
            sums[warp] = whole;
        }
        __syncthreads();
        if (!direct && warp == 0) segment_sum(part.sum, part.top);
    }
    // ---- the row's last block: its candidates ----
    if (!direct) {
        if (a.segs == 1) __syncthreads();
        else if (!last_of(a.counters + row, a.segs, &flag)) return;
    }
    Candidates* const rows = reinterpret_cast<Candidates*>(a.rows);
    Candidates& out = rows[row];
    const Key last_bits = 31 - (row - group * a.beams);
    if (looked_at) {
        const int seg0 = direct ? seg : 0, segs = direct ? 1 : a.segs;   // (direct: a segment as the row is)
        const Part* const p = parts + (int64_t)row * a.segs;
        // By all threads: the `picks` largest keys of those found, in order, and how many there are.
        auto settle = [&]() {
            __syncthreads();
            const int n = count;
            places_of(found, n, [&](int place, Key k) {
                if (place < picks) best[place] = k;
            });
            __syncthreads();
            return min(n, picks);
        };
        // The same where another look might find no room: they are the first ones that are found then.
        auto make_room = [&]() {
            const int n = settle();
            if (tid < n) found[tid] = best[tid];
            if (tid == 0) count = n;
            __syncthreads();
        };
        // A key to the found ones, by whole warps: one place after the other (with an atomic operation of each lane, 157 values of a small vocabulary took 8000 clocks).
        auto add = [&](bool take, Key key) {
            const unsigned who = __ballot_sync(0xffffffffu, take);
            if (who == 0) return;
            int to = 0;
            if (lane == 0) to = atomicAdd(&count, __popc(who));
            to = __shfl_sync(0xffffffffu, to, 0) + __popc(who & ((1u << lane) - 1u));
            if (take) found[to] = key;
        };
        constexpr int AHEAD = 6;   // loads in flight; so many keys of each thread may come before the next look at how many there are
        static_assert(MOST_PICKS + 2 * AHEAD * THREADS <= ROOM, "room");
        // each thread's best key; the segments' largest values and sums
        unsigned mine = 0, k[AHEAD];   // (k: of the segments s0 ..)
        auto keys_from = [&](int s0) {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) k[j] = !direct && s0 + j < segs ? __ldcg(&p[s0 + j].key[tid]) : 0u;
        };
        keys_from(0);
        if (direct) k[0] = own;
        unsigned top = !direct && lane < segs ? __ldcg(&p[lane].top) : 0u;
        const unsigned top0 = top;
        const double y0 = !direct && lane < segs ? __ldcg(&p[lane].sum) : 0.;
        for (int s = lane + 32; s < segs; s += 32) top = max(top, __ldcg(&p[s].top));   // (each warp for itself)
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) mine = max(mine, k[j] >> 16);
#pragma unroll 4
        for (int s = AHEAD; s < segs; ++s) mine = max(mine, __ldcg(&p[s].key[tid]) >> 16);
        top = __reduce_max_sync(0xffffffffu, top);
        const double most = value_of(top);
        // Twice `picks` of these, a quarter of that many the largest ones of each warp: no share whose code is below the `picks`-th of them can be among the best.
        const int each = (picks + 3) / 4;
        unsigned left = mine > NO_VALUE ? mine << 8 | tid : 0u;
#pragma unroll 1
        for (int i = 0; i < each; ++i) {
            const unsigned m = __reduce_max_sync(0xffffffffu, left);
            if (left == m) left = 0;
            if (lane == i) best_of[warp * each + i] = m;
        }
        if (tid == 0) count = 0, bar = 0u;
        __syncthreads();
        // (those of threads without values are 0, and so may be the picks-th: no bar)
        places_of(best_of, WARPS * each, [&](int place, Key k) {
            if (place == picks - 1 && k != 0) bar = (unsigned)(k >> 8);
        });
        __syncthreads();
        Key least = (Key)bar << 32;
#pragma unroll 1
        for (int s0 = 0; s0 < segs; s0 += AHEAD) {
            if (s0) keys_from(s0);
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const Key key = (Key)(k[j] >> 16) << 32 | (0xFFFFFFFFu - (unsigned)((seg0 + s0 + j) * a.per_seg + (int)(0xFFFFu - (k[j] & 0xFFFFu))));
                add(k[j] != 0 && key >= least, key);
            }
            if (s0 + AHEAD >= segs) break;
            __syncthreads();
            if (count > ROOM - AHEAD * THREADS) {   // (equal values)
                make_room();
                least = best[picks - 1];
            }
            __syncthreads();
        }
        // The shares' values that are not below the least of the maxima (of fewer shares than picks: all), a value to a thread; and the row's sum.
        const int shares = settle(), steps = (a.per_seg + THREADS - 1) / THREADS, values = steps * 8;
        least = shares == picks ? best[picks - 1] >> 32 << 32 : (Key)(NO_VALUE + 1) << 32;
        if (tid == 0) {
            count = 0;
            if (!direct) sums[0] = -1.;   // (without shares there are no candidates)
        }
        if (direct && shares == 0 && warp == 0) segment_sum(list.sum, list.top);
        if (tid < shares) homes[tid] = (int)(0xFFFFFFFFu - (unsigned)best[tid]);
        __syncthreads();
        // (two shares to a warp at a time)
        int home[2], stop[2] = {0, 0};
#pragma unroll 1
        for (int s0 = 0; s0 < shares; s0 += 2 * WARPS) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int share = s0 + q * WARPS + warp;
                home[q] = -1;
                if (share < shares) {
                    const int first = homes[share], s = first / a.per_seg;
                    home[q] = 8 * (s * a.per_seg + (first - s * a.per_seg) % THREADS);
                    stop[q] = min(a.vocab, 8 * (s + 1) * a.per_seg);
                }
            }
#pragma unroll 1
            for (int in0 = lane; in0 - lane < values; in0 += 32 * AHEAD) {
                uint16_t h[2][AHEAD];
                auto token_of = [&](int q, int j) { return home[q] + (in0 + 32 * j) / 8 * (8 * THREADS) + (in0 + 32 * j) % 8; };
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int j = 0; j < AHEAD; ++j) {
                        h[q][j] = 0xFC00;
                        if (home[q] >= 0 && in0 + 32 * j < values && token_of(q, j) < stop[q]) h[q][j] = x.p[token_of(q, j)];
                    }
                if (direct) {
                    if (warp == WARPS - 1 && s0 == 0 && in0 == lane) segment_sum(list.sum, list.top);
                } else if (warp == WARPS - 1 && s0 + 2 * WARPS >= shares && in0 == lane) {   // meanwhile the last warp has the row's sum
                    double sum = y0 != 0 ? top0 > NO_VALUE ? y0 * exp_of((double)value_of(top0) - most) : y0 : 0.;
#pragma unroll 1
                    for (int i = lane + 32; i < segs; i += 32) {
                        const unsigned c = __ldcg(&p[i].top);
                        const double y = __ldcg(&p[i].sum);
                        if (y != 0) sum += c > NO_VALUE ? y * exp_of((double)value_of(c) - most) : y;
                    }
#pragma unroll 1
                    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                    // (a NaN or an infinity among the values: no candidates)
                    sum = sum > 0 && sum < INFINITY && most < INFINITY ? log_of(sum) : -1.;
                    if (lane == 0) sums[0] = sum;
                }
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int j = 0; j < AHEAD; ++j) {
                        if (home[q] < 0 || in0 - lane + 32 * j >= values) break;   // (of the whole warp)
                        const unsigned c = code_of(h[q][j]);
                        const Key key = (Key)c << 32 | (0xFFFFFFFFu - (unsigned)token_of(q, j));
                        add(c > NO_VALUE && key >= least, key);
                    }
                if (s0 + 2 * WARPS >= shares && in0 - lane + 32 * AHEAD >= values) break;
                __syncthreads();
                if (count > ROOM - 2 * AHEAD * THREADS) {   // (equal values)
                    make_room();
                    least = best[picks - 1];
                }
                __syncthreads();
            }
        }
        const int n = settle();
        if (direct) {
            if (tid < picks) list.key[tid] = tid < n ? best[tid] : 0ull;
        } else if (tid < MOST_PICKS) {
            const double norm = sums[0];
            const bool there = tid < n && norm >= 0;
            const Key k = there ? best[tid] : 0;
            out.total[tid] = there ? (order_of((double)score + (((double)value_of((unsigned)(k >> 32)) - most) - norm)) & ~31ull) | last_bits : 0ull;
            out.token[tid] = (int)(0xFFFFFFFFu - (unsigned)k);
        }
    } else if (!direct && tid < MOST_PICKS) {   // one candidate of a beam that has ended, none without a score
        out.total[tid] = tid == 0 && scored ? (order_of(score) & ~31ull) | last_bits : 0ull;
        out.token[tid] = a.eos;
    }
    // ---- the group's last block: the beams' lists joined, a beam to a lane ----
    __syncthreads();   // (picks fit into a warp: the first one has written)
    const int blocks = direct ? a.beams * a.segs : a.beams;   // to come
    if (blocks > 1 && !last_of(a.counters + MOST_BEAM_ROWS + group, blocks, &flag)) return;
    if (direct) {
        join_segments(a, group, *reinterpret_cast<JoinRoom*>(found));
        return;
    }
    Candidates* const all = reinterpret_cast<Candidates*>(found);
    {
        const uint4* const from = reinterpret_cast<const uint4*>(rows + (int64_t)group * a.beams);
        for (int i = tid; i < a.beams * (int)(sizeof(Candidates) / 16); i += THREADS) reinterpret_cast<uint4*>(all)[i] = __ldcg(from + i);
    }
    __syncthreads();   // (scores and flags have been read: they may be the outputs)
    // A candidate's place: its own beam's before it, and of each other beam those that come before it.
    int there = 0;
    const int half = picks > 1 ? 1 << (31 - __clz(picks - 1)) : 0;   // (a list has up to 2 * half candidates)
#pragma unroll 1
    for (int i = tid; i < a.beams * picks; i += THREADS) {
        const int b = i / picks, j = i - b * picks;
        const Key mine = all[b].total[j];
        if (mine == 0) continue;
        ++there;
        int place = j;
#pragma unroll 2
        for (int c = 0; c < a.beams; ++c) {
            const Key* const list = all[c].total;
            int before = 0;
#pragma unroll
            for (int step = MOST_PICKS / 2; step > 0; step >>= 1)
                if (step <= half && list[before + step - 1] > mine) before += step;
            before += list[before] > mine;
            place += c == b ? 0 : before;
        }
        if (place < picks) {
            const int64_t o = (int64_t)group * picks + place;
            const int token = all[b].token[j];
            a.out_score[o] = (float)total_of(mine);
            a.out_token[o] = token;
            a.out_parent[o] = b;
            if (a.out_done) a.out_done[o] = token == a.eos;
        }
    }
    if (tid == 0) count = 0;
    __syncthreads();
    if (there) atomicAdd(&count, there);
    __syncthreads();
    if (tid >= count && tid < picks) {   // no more candidates
        const int64_t o = (int64_t)group * picks + tid;
        a.out_score[o] = -INFINITY;
        a.out_token[o] = a.out_parent[o] = -1;
        if (a.out_done) a.out_done[o] = 0;
    }
}

}  // namespace

cudaError_t launch_beam_select(const BeamSelectArgs& given, int sm_count, cudaStream_t st, bool pdl) {
    BeamSelectArgs a = given;
    beam_segments(a.groups * a.beams, a.vocab, sm_count, &a.segs, &a.per_seg);
    // Few blocks look for their segments' candidates themselves, which saves the rows' counters and a trip to the parts; of many, in several rounds, most have
    // nothing to do with that.  So / by rows, us: 1 x 4 beams of 49152, 4 picks 8.5 / 9.6; of 151936 11.4 / 13.5; 8 x 5 of 65535, 5 picks 13.8 / 16.9; 64 x 4 of 8192, 8 picks
    // 11.9 / 14.9; 100 x 4 of 1000, 4 picks 10.1 / 13.0.  Without segments there is less to save and rows' lists are joined sooner where they are long: 11 x 14 of 157, 28 picks 37 / 25.
    const int lists = a.beams * a.segs, candidates = lists * a.picks;
    const bool direct = a.groups * lists <= 4 * sm_count && lists <= DIRECT_LISTS && candidates <= (a.segs > 1 ? DIRECT_MOST : DIRECT_MOST / 8);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.groups * a.beams * a.segs));
    cfg.blockDim = dim3(THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, direct ? beam_select_kernel<true> : beam_select_kernel<false>, a);
}

// Segments of a row, in whole rounds of loads: of so many that there are some 16 blocks for each SM, and of no more vectors than have numbers of 16 bits.
// (64 groups of 8 beams of 151936 logits with some 6 / 10 / 16 / 24 / 40 blocks for each SM: 51.9 / 48.5 / 45.7 / 48.6 / 51.6 us; fewer leave SMs without work at the end, more have more
// parts to read and counters to wait for)
void beam_segments(int rows, int vocab, int sm_count, int* segs, int* per_seg) {
    const int vectors = (vocab + 7) / 8, round = THREADS * BATCH, rounds = (vectors + round - 1) / round;
    const long long n = ((long long)rounds * rows + 16 * sm_count - 1) / (16 * sm_count);
    *per_seg = (int)(n < 64 ? n : 64) * round;
    *segs = (vectors + *per_seg - 1) / *per_seg;
}

}  // namespace nnb
