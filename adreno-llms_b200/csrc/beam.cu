// Beam search's selection: the best continuations of each group of beams.
//
//   total(b, v) = score_b + ((x_bv - m_b) - log sum_w exp(x_bw - m_b))      x fp16 logits, m_b the row's maximum, all in 64 bits
//
// and of an ended beam only (b, eos) with score_b.  The largest totals come first, of equal ones the lowest beam, then the lowest token.
#include <cuda_fp16.h>

#include "kv_branch.h"
#include "ptx.cuh"

namespace nnb {
namespace {

constexpr int THREADS = 256;

struct Candidate {
    double total;
    long long at;   // beam * vocab + token; -1: none
};
__device__ __forceinline__ bool better(const Candidate& a, const Candidate& b) {
    return a.at >= 0 && (b.at < 0 || a.total > b.total || (a.total == b.total && a.at < b.at));
}

// A block for each group.  Every pick goes through all logits for the best candidate behind the one before.
__global__ void __launch_bounds__(THREADS) beam_select_kernel(const BeamSelectArgs a) {
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    __shared__ double top[MOST_BEAMS], norm[MOST_BEAMS], part[THREADS];
    __shared__ Candidate best[THREADS];
    const int tid = threadIdx.x;
    for (int g = blockIdx.x; g < a.groups; g += gridDim.x) {
        auto logit = [&](int b, int v) { return (double)__half2float(__ushort_as_half(a.logits[((int64_t)g * a.beams + b) * a.stride + v])); };
        auto ended = [&](int b) { return a.done && a.done[g * a.beams + b] != 0; };
        for (int b = 0; b < a.beams; ++b) {
            double m = -INFINITY;
            for (int v = tid; v < a.vocab; v += THREADS) m = fmax(m, logit(b, v));
            __syncthreads();
            part[tid] = m;
            __syncthreads();
            for (int i = 0; i < THREADS; ++i) m = fmax(m, part[i]);
            double s = 0;
            for (int v = tid; v < a.vocab; v += THREADS) s += exp(logit(b, v) - m);
            __syncthreads();
            part[tid] = s;
            __syncthreads();
            if (tid == 0) {
                s = 0;
                for (int i = 0; i < THREADS; ++i) s += part[i];
                top[b] = m;
                norm[b] = log(s);   // NaN where the row holds a NaN or an infinity, or nothing but -infinity: no candidates
            }
        }
        __syncthreads();
        Candidate last = {INFINITY, -1};
        for (int p = 0; p < a.picks; ++p) {
            Candidate mine = {0, -1};
            for (int b = 0; b < a.beams; ++b) {
                const double score = a.score[g * a.beams + b];
                auto offer = [&](double total, int v) {
                    const Candidate c = {total, (long long)b * a.vocab + v};
                    if (total > -INFINITY && (p == 0 || better(last, c)) && better(c, mine)) mine = c;
                };
                if (ended(b)) {
                    if (tid == 0) offer(score, a.eos);
                } else {
                    for (int v = tid; v < a.vocab; v += THREADS) offer(score + ((logit(b, v) - top[b]) - norm[b]), v);
                }
            }
            __syncthreads();
            best[tid] = mine;
            __syncthreads();
            if (tid == 0) {
                for (int i = 1; i < THREADS; ++i)
                    if (better(best[i], mine)) mine = best[i];
                best[0] = mine;
            }
            __syncthreads();
            last = best[0];
            if (tid == 0) {
                const int64_t o = (int64_t)g * a.picks + p;
                const int token = last.at < 0 ? -1 : (int)(last.at % a.vocab);
                part[p] = last.total;
                a.out_token[o] = token;
                a.out_parent[o] = last.at < 0 ? -1 : (int)(last.at / a.vocab);
            }
            if (last.at < 0) {   // no more candidates
                for (int i = p + tid; i < a.picks; i += THREADS) a.out_token[(int64_t)g * a.picks + i] = a.out_parent[(int64_t)g * a.picks + i] = -1;
                break;
            }
        }
        __syncthreads();   // (scores and flags have been read: they may be the outputs)
        if (tid < a.picks) {
            const int64_t o = (int64_t)g * a.picks + tid;
            const int token = a.out_token[o];
            a.out_score[o] = token < 0 ? -INFINITY : (float)part[tid];
            if (a.out_done) a.out_done[o] = token >= 0 && token == a.eos;
        }
        __syncthreads();
    }
}

}  // namespace

cudaError_t launch_beam_select(const BeamSelectArgs& a, cudaStream_t st, bool pdl) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.groups);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, beam_select_kernel, a);
}

}  // namespace nnb
