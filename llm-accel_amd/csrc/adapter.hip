// adapter.hip -- low-rank adapters beside a resident projection.
//
// Row r under adapter (A, B, scale) of rank R gets
//   t_j  = sat32(rnd(sum_k x_k A_jk, 4))              Q16.16, 32 bits
//   m_o  = sat32(rnd(sum_j t_j B_jo, 12))             Q16.16
//   y_o  = narrow(sum_k x_k W_ok + rnd(scale m_o, 12))
// with the projection's own exact sum and narrowing, all sums in 64 bits: a
// row without an adapter is the plain projection's bit for bit.  Each
// intermediate value keeps the 16 fraction bits of the projections'
// accumulator format, so that a small t is not lost to Q8.8 (at 8 fraction
// bits a t of 0.1 would be off by up to 2 %).
//
// The weights of the shared projection bound a call and are read once for
// all rows, by the projection's own kernels, which leave their exact sums in
// `wide`; A and B of an adapter are read once for all rows under it.  Both
// are the caller's row-major memory (adapters come and go with requests), B
// as [rank][outputs] so that a wavefront reads consecutive outputs.
#include "adapter.h"

#include "proj_common.h"

namespace llm {
namespace {

// Sum over the wavefront's lanes.
__device__ __forceinline__ int64_t wave_sum64(int64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Both int16 halves shifted right by 8.  (The word by value: a bit cast of
// an element of a vector in place has been seen to take its first element.)
__device__ __forceinline__ uint32_t high_bytes(uint32_t w) {
    const s16x2 v = __builtin_bit_cast(s16x2, w);
    return __builtin_bit_cast(uint32_t, v >> 8);
}

// Workgroup (group, j): t_j of the group's rows.  256 threads take 4 inputs
// each in turn.  Products as x (256 h + l), h and l the weight's high and
// unsigned low byte, by dot2: |x h| <= 2^22 and x l < 2^23, so the int32 sums
// of 64 inputs (16 turns) stay below 2^29 and 2^30 before they widen.
template <int NR>
__device__ __forceinline__ void adapter_in_rows(const AdapterArgs& a, const AdapterGroup& g,
                                                uint32_t j, uint32_t r0, int64_t (*red)[4]) {
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
        for (uint32_t n = 0; n < 16 && k < K; n++, k += 1024) {
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
        acc[r] = wave_sum64(acc[r]);
        if ((tid & 63) == 0) red[r0 + r][tid >> 6] = acc[r];
    }
}

__global__ __launch_bounds__(256) void adapter_in_kernel(AdapterArgs a) {
    __shared__ int64_t red[8][4];
    uint32_t j = blockIdx.x, gi = 0;  // < ranks
    while (j >= a.g[gi].rank) j -= a.g[gi++].rank;
    const AdapterGroup& g = a.g[gi];
    uint32_t r = 0;
    for (; r + 4 <= g.rows; r += 4) adapter_in_rows<4>(a, g, j, r, red);
    if (r + 2 <= g.rows) adapter_in_rows<2>(a, g, j, r, red), r += 2;
    if (r < g.rows) adapter_in_rows<1>(a, g, j, r, red);
    __syncthreads();
    if (threadIdx.x < g.rows) {
        const int64_t* v = red[threadIdx.x];
        const int64_t sum = v[0] + v[1] + v[2] + v[3];
        a.t[(size_t)g.row[threadIdx.x] * kAdapterRankMax + j] = fx_sat32(fx_rnd(sum, 4));
    }
}

// Workgroup (128 outputs, group): wavefront w takes every fourth rank from w
// on, a lane two outputs; the wavefronts' sums meet in LDS.
constexpr uint32_t kOutCols = 128;
__global__ __launch_bounds__(256) void adapter_out_kernel(AdapterArgs a) {
    __shared__ int64_t red[4][8][kOutCols];
    const AdapterGroup& g = a.g[blockIdx.y];
    const uint32_t tid = threadIdx.x, lane = tid & 63, N = a.outputs;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t n0 = blockIdx.x * kOutCols, rows = g.rows;
    const uint32_t n = n0 + 2 * lane;
    int64_t acc[8][2];
#pragma unroll
    for (int r = 0; r < 8; r++) acc[r][0] = acc[r][1] = 0;
    if (n < N) {  // N is even
        const int16_t* bp = g.b + n;
#pragma unroll 4
        for (uint32_t j = wave; j < g.rank; j += 4) {
            const uint32_t w = *(const uint32_t*)(bp + (size_t)j * N);
            const int32_t b0 = (int16_t)(w & 0xffff), b1 = (int32_t)w >> 16;
#pragma unroll
            for (int r = 0; r < 8; r++) {
                if (r >= (int)rows) break;
                const int32_t t = a.t[(size_t)g.row[r] * kAdapterRankMax + j];
                acc[r][0] += (int64_t)t * b0;
                acc[r][1] += (int64_t)t * b1;
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 8; r++) {
        if (r >= (int)rows) break;
        red[wave][r][2 * lane] = acc[r][0];
        red[wave][r][2 * lane + 1] = acc[r][1];
    }
    __syncthreads();
    for (uint32_t i = tid; i < rows * kOutCols; i += 256) {
        const uint32_t r = i / kOutCols, c = i % kOutCols, o = n0 + c;
        if (o >= N) continue;
        const size_t at = (size_t)g.row[r] * N + o;
        const int64_t s = red[0][r][c] + red[1][r][c] + red[2][r][c] + red[3][r][c];
        const int64_t more = fx_rnd((int64_t)fx_sat32(fx_rnd(s, 12)) * g.scale, 12);
        a.out[at] = narrow16(a.wide[at] + more);
    }
}

}  // namespace

hipError_t launch_adapter_in(const AdapterArgs& a, hipStream_t st) {
    if (a.ranks == 0) return hipSuccess;
    adapter_in_kernel<<<a.ranks, 256, 0, st>>>(a);
    return hipGetLastError();
}
hipError_t launch_adapter_out(const AdapterArgs& a, hipStream_t st) {
    const dim3 grid((a.outputs + kOutCols - 1) / kOutCols, a.groups);
    adapter_out_kernel<<<grid, 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace llm
