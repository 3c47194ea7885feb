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
// `wide`, while other workgroups of the same launch form x A^T; A and B of an
// adapter are read once for all rows under it.  Both are the caller's row-major
// memory (adapters come and go with requests), B as [rank][outputs] so that a
// wavefront reads consecutive outputs.  Launch boundaries are what a small call
// waits for: one row of 2,048 x 2,048 took 17.8 us in four launches (a copy of
// the row, the projection, x A^T, this one) and takes 10 in these two.
#include "adapter.h"

#include "proj_common.h"

namespace llm {
namespace {

// Workgroup (128 outputs, group): wavefront w takes every fourth rank from w
// on, a lane two outputs, sixteen ranks' loads at a time; the wavefronts' sums
// meet in LDS.  Bound by two dependent loads (t, then what B's loads left) and
// the sums' exchange: 3.8 us for one row of rank 16, 4.6 for 8 rows under
// adapters of their own of rank 64 (2.1 MB of B), 2,048 outputs each.
constexpr uint32_t kOutCols = 128, kAhead = 16;
__global__ __launch_bounds__(256) void adapter_out_kernel(AdapterArgs a) {
    __shared__ int64_t red[4][8][kOutCols];
    __shared__ int32_t ts[8][kAdapterRankMax];
    const AdapterGroup& g = a.g[blockIdx.y];
    const uint32_t tid = threadIdx.x, lane = tid & 63, N = a.outputs;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t n0 = blockIdx.x * kOutCols, rows = g.rows, rank = g.rank;
    const uint32_t n = n0 + 2 * lane;
    // the projection's sums of this thread's outputs: column tid % 128, rows
    // tid / 128, + 2, ..
    const uint32_t c = tid % kOutCols, o = n0 + c;
    int64_t base[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) {
        const uint32_t r = tid / kOutCols + 2 * i;
        base[i] = r < rows && o < N ? a.wide[(size_t)g.row[r] * N + o] : 0;
    }
    const int16_t* bp = g.b + n;
    uint32_t bw[kAhead];
    auto b_load = [&](uint32_t j0) {
#pragma unroll
        for (uint32_t u = 0; u < kAhead; u++) {
            const uint32_t j = j0 + 4 * u + wave;
            bw[u] = j < rank && n < N ? *(const uint32_t*)(bp + (size_t)j * N) : 0;  // N is even
        }
    };
    b_load(0);
    for (uint32_t r = 0; r < rows; r++)
        for (uint32_t j = tid; j < rank; j += 256)
            ts[r][j] = a.t[(size_t)g.row[r] * kAdapterRankMax + j];
    int64_t acc[8][2];
#pragma unroll
    for (int r = 0; r < 8; r++) acc[r][0] = acc[r][1] = 0;
    __syncthreads();
    for (uint32_t j0 = 0; j0 < rank; j0 += 4 * kAhead) {
        if (j0) b_load(j0);
#pragma unroll
        for (uint32_t u = 0; u < kAhead; u++) {
            const uint32_t j = j0 + 4 * u + wave;
            if (j >= rank) break;
            const int32_t b0 = (int16_t)(bw[u] & 0xffff), b1 = (int32_t)bw[u] >> 16;
#pragma unroll
            for (int r = 0; r < 8; r++) {
                if (r >= (int)rows) break;
                acc[r][0] += (int64_t)ts[r][j] * b0;
                acc[r][1] += (int64_t)ts[r][j] * b1;
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
    if (o >= N) return;
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) {
        const uint32_t r = tid / kOutCols + 2 * i;
        if (r >= rows) break;
        const int64_t s = red[0][r][c] + red[1][r][c] + red[2][r][c] + red[3][r][c];
        const int64_t more = fx_rnd((int64_t)fx_sat32(fx_rnd(s, 12)) * g.scale, 12);
        a.out[(size_t)g.row[r] * N + o] = narrow16(base[i] + more);
    }
}

}  // namespace

hipError_t launch_adapter_out(const AdapterArgs& a, hipStream_t st) {
    const dim3 grid((a.outputs + kOutCols - 1) / kOutCols, a.groups);
    adapter_out_kernel<<<grid, 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace llm
