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

// Column j of A's product for NR of the group's rows.  NT threads take 4
// inputs each in turn.  Products as x (256 h + l), h and l the weight's high
// and unsigned low byte, by dot2: |x h| <= 2^22 and x l < 2^23, so the int32
// sums of 64 inputs (16 turns) stay below 2^29 and 2^30 before they widen.
template <int NR, int NT>
__device__ __forceinline__ void adapter_in_rows(const AdapterArgs& a, const AdapterGroup& g,
                                                uint32_t j, uint32_t r0,
                                                int64_t (*red)[NT / 64]) {
    const uint32_t tid = threadIdx.x, K = a.inputs;
    const int16_t* ap = g.a + (size_t)j * K;
    const int16_t* xp[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) xp[r] = a.x + (size_t)g.row[r0 + r] * K;
    int64_t acc[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) acc[r] = 0;
    for (uint32_t k = 4 * tid; k < K;) {
        int32_t hi[NR], lo[NR];
#pragma unroll
        for (int r = 0; r < NR; r++) hi[r] = lo[r] = 0;
#pragma unroll 2
        for (uint32_t n = 0; n < 16 && k < K; n++, k += 4 * NT) {
            const v2u w = *(const v2u*)(ap + k);
            const uint32_t h0 = high_bytes(w.x), h1 = high_bytes(w.y);
            const uint32_t l0 = w.x & 0x00ff00ffu, l1 = w.y & 0x00ff00ffu;
#pragma unroll
            for (int r = 0; r < NR; r++) {
                const v2u x = *(const v2u*)(xp[r] + k);
                hi[r] = dot2(h0, x.x, hi[r]);
                lo[r] = dot2(l0, x.x, lo[r]);
                hi[r] = dot2(h1, x.y, hi[r]);
                lo[r] = dot2(l1, x.y, lo[r]);
            }
        }
#pragma unroll
        for (int r = 0; r < NR; r++) acc[r] += 256 * (int64_t)hi[r] + lo[r];
    }
#pragma unroll
    for (int r = 0; r < NR; r++) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) acc[r] += __shfl_xor(acc[r], o, 64);
        if ((tid & 63) == 0) red[r0 + r][tid >> 6] = acc[r];
    }
}

// Workgroup `block` of a.ranks: one column j of one group's A^T.
template <int NT>
__device__ __forceinline__ void adapter_in_block(const AdapterArgs& a, uint32_t block) {
    __shared__ int64_t red[8][NT / 64];
    uint32_t j = block, gi = 0;
    while (j >= a.g[gi].rank) j -= a.g[gi++].rank;
    const AdapterGroup& g = a.g[gi];
    uint32_t r = 0;
    for (; r + 4 <= g.rows; r += 4) adapter_in_rows<4, NT>(a, g, j, r, red);
    if (r + 2 <= g.rows) adapter_in_rows<2, NT>(a, g, j, r, red), r += 2;
    if (r < g.rows) adapter_in_rows<1, NT>(a, g, j, r, red);
    __syncthreads();
    if (threadIdx.x < g.rows) {
        int64_t sum = 0;
#pragma unroll
        for (int w = 0; w < NT / 64; w++) sum += red[threadIdx.x][w];
        a.t[(size_t)g.row[threadIdx.x] * kAdapterRankMax + j] = fx_sat32(fx_rnd(sum, 4));
    }
}

}  // namespace
}  // namespace llm
