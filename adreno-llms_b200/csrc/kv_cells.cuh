// Reading and writing cells of the key/value cache.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <climits>

#include "attention.h"
#include "ptx.cuh"

namespace nnb {

// Two e4m3 codes (low byte first) as half2, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
    return r;
}
// Four 8-bit codes of one word -> two half2, exact.
template <int FMT>
__device__ __forceinline__ void codes_to_half2x2(uint32_t w, uint32_t& h01, uint32_t& h23) {
    if (FMT == KV_INT8) {
        int8x4_to_half2x2(w, h01, h23);
    } else {
        h01 = e4m3x2_to_half2(w & 0xFFFFu);
        h23 = e4m3x2_to_half2(w >> 16);
    }
}
__device__ __forceinline__ float2 half2_floats(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float half_float(uint16_t h) { return __half2float(__ushort_as_half(h)); }
// From here on a value is an infinity as fp16.  (The attention's weights are rounded for their product with the values and not in their sum, so that a
// result may pass the largest value by 2^-11 of it: such a row is computed once more, with weights of 32 bits.)
constexpr float HALF_END = 65520.f;
__device__ __forceinline__ uint32_t floats_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The scale of a row whose largest magnitude is `most`: the smallest fp16 s with s * Q >= most, Q the largest code (the product of 11 and
// at most 9 bits is exact in 32), so that no code is cut off; one less
// where s * Q is no fp16 value any more (rows that reach 65504, which must not read back as infinite).  1 for a row of zeros; NaN where the row holds an infinity or a NaN: such a
// row reads back as NaN as a whole.
__device__ __forceinline__ uint16_t row_scale(float most, float Q) {
    if (!(most <= 65504.f)) return 0x7FFF;
    if (most == 0.f) return 0x3C00;
    uint16_t s = __half_as_ushort(__float2half_rn(most / Q));
    if (half_float(s) * Q < most) ++s;
    if (half_float(s) * Q > 65504.f) --s;
    return s;
}

// Where a row of a call belongs.  By a whole warp.
struct RowPlace {
    bool none;   // behind the last sequence, or before the first
    bool bad;    // its sequence's numbers are out of range
    int seq, pos;
};
__device__ __forceinline__ RowPlace place_of_row(const KvSeqs& s, int r) {
    const int lane = threadIdx.x & 31;
    RowPlace p;
    p.seq = 0;   // how many sequences end at or before it
    for (int i0 = 0; i0 < s.num_seqs; i0 += 32) {
        const int i = i0 + lane;
        const unsigned before = __ballot_sync(0xffffffffu, i < s.num_seqs && s.row_start[i + 1] <= r);
        p.seq += __popc(before);
        if (before != 0xffffffffu) break;   // (they ascend)
    }
    p.none = p.seq >= s.num_seqs || (p.seq == 0 && r < s.row_start[0]);
    p.bad = false;
    p.pos = 0;
    if (p.none) return p;
    const SeqExtent e = seq_extent(s.row_start[p.seq], s.row_start[p.seq + 1], s.kv_len[p.seq], s.num_rows, s.max_len);
    p.pos = e.len - (e.row1 - r);
    p.bad = e.bad || p.pos < 0 || r < e.row0 || r >= e.row1;
    return p;
}
// The same with one trip to memory for each 64 sequences: a lane has the numbers of one in either half of them.  (For writes: 64 rows of 48 heads of 128 dims, e4m3, 3.2 us by
// the one above, 3.0 by this; reads of 65536 rows 217 and 222.)
__device__ __forceinline__ RowPlace place_of_row_soon(const KvSeqs& s, int r) {
    const int lane = threadIdx.x & 31;
    RowPlace p;
    p.seq = p.pos = 0;
    p.none = true;
    p.bad = false;
    for (int i0 = 0; i0 < s.num_seqs; i0 += 64) {
        int start[2], end[2], len[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const int i = i0 + 32 * g + lane, j = min(i, s.num_seqs - 1);
            start[g] = s.row_start[j];
            end[g] = s.row_start[j + 1];
            len[g] = s.kv_len[j];
            if (i >= s.num_seqs) end[g] = INT_MAX;
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const unsigned before = __ballot_sync(0xffffffffu, end[g] <= r);   // sequences that end at or before it (they ascend)
            if (before == 0xffffffffu) continue;
            const int from = __popc(before), first = __shfl_sync(0xffffffffu, start[g], from), last = __shfl_sync(0xffffffffu, end[g], from), kv_len = __shfl_sync(0xffffffffu, len[g], from);
            p.seq = i0 + 32 * g + from;
            p.none = p.seq >= s.num_seqs || (p.seq == 0 && r < first);
            if (p.none) return p;
            const SeqExtent e = seq_extent(first, last, kv_len, s.num_rows, s.max_len);
            p.pos = e.len - (e.row1 - r);
            p.bad = e.bad || p.pos < 0 || r < e.row0 || r >= e.row1;
            return p;
        }
    }
    return p;
}

}  // namespace nnb
