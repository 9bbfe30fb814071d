// Beam search's selection: the best continuations of each group of beams.
//
//   total(b, v) = score_b + ((x_bv - m_b) - log sum_w exp(x_bw - m_b))      x fp16 logits, m_b the row's maximum
//
// and of an ended beam only (b, eos) with score_b.  The largest totals come first, of equal ones the lowest beam, then the lowest token.
//
// Bound by the logits' bytes, each read once.  A row is cut into segments, a block each; a thread has up to CHUNK vectors of 8 values of its segment and
// keeps their maximum, where it first was, and the sum of exponentials behind it.  The row's best `picks` values lie in those threads' shares whose
// maxima are the `picks` best ones: every other share has `picks` values before all of its own.  So no value needs a place in a list while the
// logits stream by, whatever their order; the last block of a group reads the few shares again that matter (picks * CHUNK vectors of a row).
//
// Within a row the fp16 values and the tokens decide, exactly.  Across rows the totals do, in 64 bits.  Exponentials are taken of differences to the
// thread's maximum (exact), in 32 bits: a maximum is exactly 1, the others are 2^-22 off at most, and so is the sum; a row of 151936 values of N(0, 2.5) has a sum that is some
// 2^-28 off, its errors being different for each value.  Everything depends on differences alone: rows that are shifted against each other
// give the same logarithms.
#include <cuda_fp16.h>

#include "kv_branch.h"
#include "ptx.cuh"

namespace nnb {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32, BATCH = 4;
constexpr int CHUNK = 8;                    // vectors of a thread at most
constexpr unsigned NO_VALUE = 0x03FFu;      // the code of -infinity

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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

// 32 keys of a warp, the largest first
template <class Key>
__device__ __forceinline__ Key larger(Key a, Key b) { return a > b ? a : b; }
template <class Key>
__device__ __forceinline__ Key smaller(Key a, Key b) { return a > b ? b : a; }
template <class Key>
__device__ __forceinline__ Key ordered(Key x) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int d = size >> 1; d > 0; d >>= 1) {
            const Key y = __shfl_xor_sync(0xffffffffu, x, d);
            x = ((lane & d) == 0) == ((lane & size) == 0 || size == 32) ? larger(x, y) : smaller(x, y);
        }
    return x;
}
// The 32 largest of two such lists
template <class Key>
__device__ __forceinline__ Key merged(Key a, Key b) {
    const int lane = threadIdx.x & 31;
    a = larger(a, __shfl_sync(0xffffffffu, b, 31 - lane));
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const Key y = __shfl_xor_sync(0xffffffffu, a, d);
        a = (lane & d) == 0 ? larger(a, y) : smaller(a, y);
    }
    return a;
}
template <class Key, class At>
__device__ __forceinline__ Key merged8(At&& at) {
    Key x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = at(i);
#pragma unroll
    for (int n = 4; n > 0; n >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) x[i] = merged(x[i], x[i + n]);
    return x[0];
}

// A row of logits as vectors of 8 tokens, wherever the row begins (so that equal rows are added up in the same order and give the same bits).
// Behind the row's end there is -infinity.
struct Row {
    const uint16_t* p;
    int vocab;
    __device__ __forceinline__ Row(const uint16_t* row, int v) : p(row), vocab(v) {}
    __device__ __forceinline__ int vectors() const { return (vocab + 7) / 8; }
    __device__ __forceinline__ uint4 load(int i) const {
        const int off = (int)(reinterpret_cast<uintptr_t>(p) & 15);   // the same for all of the row's vectors
        const uint16_t* const at = p + (int64_t)8 * i;
        uint4 x;
        if (off == 0 && 8 * i + 8 <= vocab) {
            asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(at));
        } else if (off != 0 && i > 0 && 8 * i + 16 - off / 2 <= vocab) {   // two pieces at 16-byte boundaries; the second is the next thread's first
            const uint4* const two = reinterpret_cast<const uint4*>(at - off / 2);
            const uint4 a = __ldg(two), b = __ldg(two + 1);
            uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
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
            x = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = 8 * i + 2 * j;
                w[j] = (t < vocab ? at[2 * j] : 0xFC00u) | (uint32_t)(t + 1 < vocab ? at[2 * j + 1] : 0xFC00u) << 16;
            }
            x = make_uint4(w[0], w[1], w[2], w[3]);
        }
        return x;
    }
};
__device__ __forceinline__ __half2 as_half2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }
__device__ __forceinline__ float most_of(const uint4& x) {
    const __half2 m = __hmax2(__hmax2(as_half2(x.x), as_half2(x.y)), __hmax2(as_half2(x.z), as_half2(x.w)));
    return __half2float(__hmax(__low2half(m), __high2half(m)));
}

struct Part {   // of a segment: the sum of exponentials behind its largest value
    double sum;
    unsigned keys[MOST_PICKS];   // code << 16 | 0xFFFF - vector in the segment: its threads' largest values, in order
};
static_assert(sizeof(Part) == BEAM_PART_BYTES, "workspace");

__global__ void __launch_bounds__(THREADS) beam_select_kernel(const BeamSelectArgs a) {
    __shared__ unsigned lists[WARPS][32];
    __shared__ double sums[WARPS];
    __shared__ double totals[MOST_BEAMS][MOST_PICKS];   // of each beam its best candidates, in order
    __shared__ int tokens[MOST_BEAMS][MOST_PICKS], flag;
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x / a.segs, seg = blockIdx.x - row * a.segs, group = row / a.beams;
    // A beam that has ended, or has no score, is not looked at.
    auto looked_at = [&](int r) { return !(a.done && a.done[r] != 0) && a.score[r] > -INFINITY; };
    Part* const parts = reinterpret_cast<Part*>(a.parts);
    if (looked_at(row)) {
        const Row x(a.logits + (int64_t)row * a.stride, a.vocab);
        const int begin = seg * a.per_seg, end = min(x.vectors(), begin + a.per_seg);
        float most = -INFINITY, sum = 0.f, rest = 0.f;   // (rest: what rounding has taken from the sum)
        int at = 0;
        for (int i0 = begin + tid; i0 < end; i0 += THREADS * BATCH) {
            uint4 v[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) v[j] = i0 + j * THREADS < end ? x.load(i0 + j * THREADS) : make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u);
            float m[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) m[j] = most_of(v[j]);
            const float up = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
            if (up > most) {
                const float f = ex2((most - up) * 1.4426950408889634f);
                sum *= f;
                rest *= f;
                most = up;
#pragma unroll
                for (int j = BATCH - 1; j >= 0; --j)
                    if (m[j] == up) at = i0 + j * THREADS - begin;
            }
            const float ref = most == -INFINITY ? 0.f : most;
            float s[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
                float e[8];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float2 y = __half22float2(as_half2(w[q]));
                    e[2 * q] = ex2((y.x - ref) * 1.4426950408889634f);
                    e[2 * q + 1] = ex2((y.y - ref) * 1.4426950408889634f);
                }
                s[j] = ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
            }
            const float more = (s[0] + s[1]) + (s[2] + s[3]), whole = __fadd_rn(sum, more), back = __fsub_rn(whole, sum);   // the sum's error (D. Knuth, The Art of Computer Programming 2, 4.2.2)
            rest += __fadd_rn(__fsub_rn(sum, __fsub_rn(whole, back)), __fsub_rn(more, back));
            sum = whole;
        }
        const unsigned code = code_of(__half_as_ushort(__float2half_rn(most)));
        const unsigned list = ordered(code > NO_VALUE ? code << 16 | (0xFFFFu - at) : 0u);
        lists[warp][lane] = list;
        __syncthreads();
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) top = larger(top, lists[i][0]);
        double mine = 0;
        if (sum != 0.f) mine = ((double)sum + (double)rest) * exp((double)most - (double)value_of(top >> 16));
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
        if (lane == 0) sums[warp] = mine;
        Part& part = parts[blockIdx.x];
        if (warp == 0) {
            const unsigned best = merged8<unsigned>([&](int i) { return lists[i][lane]; });
            if (lane < a.picks) part.keys[lane] = best;
        }
        __syncthreads();
        if (tid == 0) {
            double s = 0;
#pragma unroll
            for (int i = 0; i < WARPS; ++i) s += sums[i];
            part.sum = s;
        }
    }
    // ---- the group's last block has the parts of all of its rows ----
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        const bool last = atomicAdd(a.counters + group, 1u) == (unsigned)(a.beams * a.segs - 1);
        if (last) a.counters[group] = 0u;
        flag = last;
    }
    __syncthreads();
    if (!flag) return;
    __threadfence();
    for (int b = warp; b < a.beams; b += WARPS) {
        const int r = group * a.beams + b;
        double total = -INFINITY;
        int token = -1;
        if (looked_at(r)) {
            const Row x(a.logits + (int64_t)r * a.stride, a.vocab);
            const Part* const p = parts + (int64_t)r * a.segs;
            // the shares with the best values, and the row's largest one
            using Key = unsigned long long;
            Key best = 0;
            for (int s0 = 0; s0 < a.segs; s0 += 8) {
                const Key more = merged8<Key>([&](int i) {
                    const int s = s0 + i;
                    const unsigned k = s < a.segs && lane < a.picks ? __ldcg(&p[s].keys[lane]) : 0u;
                    return k ? (Key)(k >> 16) << 32 | (0xFFFFFFFFu - (unsigned)(s * a.per_seg + (0xFFFF - (int)(k & 0xFFFFu)))) : (Key)0;
                });
                best = s0 ? merged(best, more) : more;
            }
            const float most = value_of((unsigned)(__shfl_sync(0xffffffffu, best, 0) >> 32));
            double sum = 0;
            for (int s = lane; s < a.segs; s += 32) {
                const unsigned k = __ldcg(&p[s].keys[0]);
                const double y = __ldcg(&p[s].sum);
                if (y != 0) sum += k ? y * exp((double)value_of(k >> 16) - (double)most) : y;
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (sum > 0 && sum < INFINITY && most < INFINITY) {
                // their values that are not below the least of these maxima, one after the other into a list
                const int shares = __popc(__ballot_sync(0xffffffffu, lane < a.picks && best != 0)), steps = (a.per_seg + THREADS - 1) / THREADS;
                const unsigned last = (unsigned)(__shfl_sync(0xffffffffu, best, shares - 1) >> 32), least = shares == a.picks ? last : 0u;   // (fewer shares: all of their values)
                Key list = 0;
                for (int i0 = 0; i0 < shares * steps; i0 += 32) {
                    const int i = i0 + lane, from = i / steps;
                    const int home = (int)(0xFFFFFFFFu - (unsigned)__shfl_sync(0xffffffffu, best, from & 31)), s = home / a.per_seg;
                    const int vec = s * a.per_seg + (home - s * a.per_seg) % THREADS + (i - from * steps) * THREADS;
                    const bool there = i < shares * steps && vec < min(x.vectors(), (s + 1) * a.per_seg);
                    const uint4 v = there ? x.load(vec) : make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u);
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll 1
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t two = e < 4 ? e < 2 ? w[0] : w[1] : e < 6 ? w[2] : w[3];
                        const unsigned code = code_of((uint16_t)(e & 1 ? two >> 16 : two));
                        const Key key = (Key)code << 32 | (0xFFFFFFFFu - (unsigned)(8 * vec + e));
                        for (unsigned left = __ballot_sync(0xffffffffu, code >= least && code > NO_VALUE); left; left &= left - 1) {
                            const Key k = __shfl_sync(0xffffffffu, key, __ffs(left) - 1), before = __shfl_up_sync(0xffffffffu, list, 1);
                            const int place = __popc(__ballot_sync(0xffffffffu, list > k));
                            if (lane >= place) list = lane == place ? k : before;
                        }
                    }
                }
                if (list != 0 && lane < a.picks) {
                    token = (int)(0xFFFFFFFFu - (unsigned)list);
                    total = (double)a.score[r] + (((double)value_of((unsigned)(list >> 32)) - (double)most) - log(sum));
                }
            }
        } else if (lane == 0 && a.score[r] > -INFINITY) {   // it has ended
            total = a.score[r];
            token = a.eos;
        }
        if (lane < a.picks) {
            totals[b][lane] = total;
            tokens[b][lane] = token;
        }
    }
    __syncthreads();   // (scores and flags have been read: they may be the outputs)
    if (warp != 0) return;
    // ---- the beams' lists joined: a beam to a lane ----
    int next = 0;   // candidates of this lane's beam that have been taken
    for (int p = 0; p < a.picks; ++p) {
        const bool there = lane < a.beams && next < a.picks && tokens[lane][next] >= 0;
        double most = there ? totals[lane][next] : -INFINITY;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) most = fmax(most, __shfl_xor_sync(0xffffffffu, most, d));
        const unsigned hit = __ballot_sync(0xffffffffu, there && totals[lane][next] == most);
        const int b = __ffs(hit) - 1;
        const int64_t o = (int64_t)group * a.picks + p;
        if (lane == (hit ? b : 0)) {
            const int token = hit ? tokens[lane][next] : -1;
            a.out_score[o] = hit ? (float)most : -INFINITY;
            a.out_token[o] = token;
            a.out_parent[o] = b;
            if (a.out_done) a.out_done[o] = hit && token == a.eos;
            if (hit) ++next;
        }
    }
}

}  // namespace

cudaError_t launch_beam_select(const BeamSelectArgs& given, int sm_count, cudaStream_t st, bool pdl) {
    BeamSelectArgs a = given;
    beam_segments(a.groups * a.beams, a.vocab, sm_count, &a.segs, &a.per_seg);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.groups * a.beams * a.segs));
    cfg.blockDim = dim3(THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, beam_select_kernel, a);
}

// Segments of a row: as many as its vectors need at CHUNK to a thread, more where the rows alone would leave SMs idle, but none with less than a vector for
// each thread.
void beam_segments(int rows, int vocab, int sm_count, int* segs, int* per_seg) {
    const int vectors = (vocab + 7) / 8, least = (vectors + THREADS * CHUNK - 1) / (THREADS * CHUNK), most = (vectors + THREADS - 1) / THREADS;
    int n = sm_count / rows;
    n = n < least ? least : n > most ? most : n;
    *per_seg = (vectors + n - 1) / n;
    *segs = (vectors + *per_seg - 1) / *per_seg;
}

}  // namespace nnb
