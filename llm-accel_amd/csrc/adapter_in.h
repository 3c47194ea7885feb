// adapter_in.h -- x A^T of the adapters' rows, by workgroups of the launch that
// forms the projection's exact sums (internal to the library).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "adapter.h"
#include "attn_common.h"
#include "fixed_point.h"

namespace llm {
namespace {

// Both int16 halves shifted right by 8.  (The word by value: a bit cast of
// an element of a vector in place has been seen to take its first element.)
__device__ __forceinline__ uint32_t high_bytes(uint32_t w) {
    const s16x2 v = __builtin_bit_cast(s16x2, w);
    return __builtin_bit_cast(uint32_t, v >> 8);
}

// Bound by the launch it is part of: 8 rows under adapters of their own of rank
// 64 beside 11,008 x 2,048 weights (11.3 MB of A, 33.8 of weights) 16.0 us,
// 2.8 TB/s; the projection alone about 12.  256 threads to a column: 11,008
// inputs in 11 turns.
constexpr uint32_t kInThreads = 256;  // of one column

// Column j of A's product for NR of the group's rows, by 256 threads (t of
// them) that take 4 inputs each in turn, up to U turns' loads at a time.
// Products as x (256 h + l), h and l the weight's high and unsigned low byte,
// by dot2: |x h| <= 2^22 and x l < 2^23, so the int32 sums of 64 inputs (16
// turns) stay below 2^29 and 2^30 before they widen.
template <int NR>
__device__ __forceinline__ void adapter_in_rows(const AdapterArgs& a, const AdapterGroup& g,
                                                uint32_t j, uint32_t r0, uint32_t t,
                                                int64_t (*red)[4]) {
    constexpr uint32_t U = NR == 1 ? 4 : 2;
    static_assert(U <= 16, "turns before the sums widen");
    const uint32_t K = a.inputs;
    const int16_t* ap = g.a + (size_t)j * K;
    const int16_t* xp[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) xp[r] = a.x + (size_t)g.row[r0 + r] * K;
    int64_t acc[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) acc[r] = 0;
#pragma unroll 1
    for (uint32_t k0 = 4 * t; k0 < K; k0 += 4 * kInThreads * U) {
        v2u w[U], x[NR][U];
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            // turns past the last repeat input 0, with no weight
            const uint32_t k = k0 + 4 * kInThreads * u, at = k < K ? k : 0;
            w[u] = *(const v2u*)(ap + at);
            if (k >= K) w[u] = v2u{0, 0};
#pragma unroll
            for (int r = 0; r < NR; r++) x[r][u] = *(const v2u*)(xp[r] + at);
        }
#pragma unroll
        for (int r = 0; r < NR; r++) {
            int32_t hi = 0, lo = 0;
#pragma unroll
            for (uint32_t u = 0; u < U; u++) {
                hi = dot2(high_bytes(w[u].x), x[r][u].x, hi);
                lo = dot2(w[u].x & 0x00ff00ffu, x[r][u].x, lo);
                hi = dot2(high_bytes(w[u].y), x[r][u].y, hi);
                lo = dot2(w[u].y & 0x00ff00ffu, x[r][u].y, lo);
            }
            acc[r] += 256 * (int64_t)hi + lo;
        }
    }
#pragma unroll
    for (int r = 0; r < NR; r++) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) acc[r] += __shfl_xor(acc[r], o, 64);
        if ((t & 63) == 0) red[r0 + r][t >> 6] = acc[r];
    }
}

// Workgroup `block` of NT threads: the next NT / 256 columns.
template <int NT>
__device__ __forceinline__ void adapter_in_block(const AdapterArgs& a, uint32_t block) {
    constexpr uint32_t C = NT / kInThreads;
    __shared__ int64_t red[C][8][4];
    const uint32_t c = __builtin_amdgcn_readfirstlane(threadIdx.x / kInThreads);
    const uint32_t t = threadIdx.x % kInThreads, column = block * C + c;
    const bool there = column < a.ranks;
    // the last group that starts at or before the column (one of rank 0 before
    // it starts there too)
    uint32_t gi = 0;
#pragma unroll
    for (uint32_t i = 1; i < 8; i++) gi += there && column >= a.start[i];
    const uint32_t j = there ? column - a.start[gi] : 0;
    const AdapterGroup& g = a.g[gi];
    if (there) {
        uint32_t r = 0;
        for (; r + 4 <= g.rows; r += 4) adapter_in_rows<4>(a, g, j, r, t, red[c]);
        if (r + 2 <= g.rows) adapter_in_rows<2>(a, g, j, r, t, red[c]), r += 2;
        if (r < g.rows) adapter_in_rows<1>(a, g, j, r, t, red[c]);
    }
    __syncthreads();
    if (there && t < g.rows) {
        const int64_t* v = red[c][t];
        a.t[(size_t)g.row[t] * kAdapterRankMax + j] =
            fx_sat32(fx_rnd(v[0] + v[1] + v[2] + v[3], 4));
    }
}

}  // namespace
}  // namespace llm
