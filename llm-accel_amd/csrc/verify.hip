// verify.hip -- next-token probabilities from the LM head's scores, and the
// verification of drafted tokens against them.
//
// Mathematics (all whole numbers, every step exact or one stated rounding,
// sums in 64 bits and so independent of their order):
//   scores s_v with 20 fraction bits, c = log2(e) / temperature with 24;
//   y_v = floor(min(s_max - s_v, 2^31) c / 2^24), octaves below the largest
//         with 20 fraction bits (temperature <= 64: what the clamp cuts is
//         below 2^-31 of the largest and weighs 0 either way);
//   w_v = floor(floor(E1[y / 2^10 mod 2^10] E2[y mod 2^10] / 2^30) / 2^n),
//         n = floor(y / 2^20), E1[i] = 2^(-i / 2^10) and E2[i] = 2^(-i /
//         2^20) rounded to 30 fraction bits: 2^-y within 2^-20 ln 2 of its
//         value (the rounding of y) plus 2^-30 of the largest;
//   P_v = floor(2^32 w_v / sum w), Q0.32, at most 2^32 - 1.
// A draft x of a row is taken iff u Q_x < 2^32 P_x (u 32 bits, uniform): with
// probability min(1, P / Q).  At a request's first row whose draft is not
// taken the next token is drawn from max(P - Q, 0) -- at the row after the
// last draft, or where that is 0 everywhere, from P -- by R = its sum, t =
// floor(u R / 2^32) and the first token whose running sum passes t.
//
// The table of the LM head bounds a call (622 MB for 151,936 x 2,048: the
// scores' pass reads it once and writes 8 bytes per score); what follows are
// two short passes over the scores, one workgroup per 2,048 of them and row
// (or request): the weights' sums, then the probabilities or the draws, the
// last workgroup of a request to arrive drawing its token.
#include "verify.h"

#include "coherent.h"
#include "kernels.h"

namespace llm {
namespace {

struct Exp2 {
    uint32_t hi[kExp2Entries], lo[kExp2Entries];
};
__device__ __forceinline__ void exp2_load(const uint32_t* t, Exp2& e) {
    for (uint32_t i = threadIdx.x; i < kExp2Entries / 4; i += 256) {
        ((uint4*)e.hi)[i] = ((const uint4*)t)[i];
        ((uint4*)e.lo)[i] = ((const uint4*)(t + kExp2Entries))[i];
    }
}

// w_v of a score `below` (>= 0) the row's largest.
__device__ __forceinline__ uint32_t weight(const Exp2& e, int64_t below, uint32_t c) {
    const uint32_t d = below > (int64_t)1 << 31 ? 1u << 31 : (uint32_t)below;
    const uint64_t y = ((uint64_t)d * c) >> 24;  // < 2^39
    const uint64_t n = y >> 20;
    if (n > 30) return 0;
    const uint32_t i = (uint32_t)y;
    return (uint32_t)(((uint64_t)e.hi[(i >> 10) & 1023] * e.lo[i & 1023]) >> 30) >> (uint32_t)n;
}

// floor(2^32 w / z) for w <= z, at most 2^32 - 1: the quotient in double
// precision (w 2^32 is exact there, the product within 2^-19 of the quotient,
// which is at most 2^32) and its remainder's sign.
__device__ __forceinline__ uint32_t prob32(uint32_t w, uint64_t z, double inv) {
    if (w == 0) return 0;
    const uint64_t num = (uint64_t)w << 32;
    uint64_t q = (uint64_t)((double)num * inv);
    int64_t r = (int64_t)(num - q * z);
    if (r < 0)
        q--;
    else if (r >= (int64_t)z)
        q++;
    return q > 0xffffffffu ? 0xffffffffu : (uint32_t)q;
}

__device__ __forceinline__ unsigned long long wave_sum64(unsigned long long v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// Sum over the workgroup's 256 threads, uniform; red: 4 words.
__device__ __forceinline__ unsigned long long block_sum64(unsigned long long v,
                                                          unsigned long long* red) {
    v = wave_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
}

// Sum of v over the threads below this one; red: 4 words.
__device__ __forceinline__ unsigned long long block_below64(unsigned long long v,
                                                            unsigned long long* red) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned long long s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned long long u = __shfl_up(s, o, 64);
        if ((int)lane >= o) s += u;
    }
    __syncthreads();
    if (lane == 63) red[wave] = s;
    __syncthreads();
    for (uint32_t w = 0; w < wave; w++) s += red[w];
    return s - v;
}

// Workgroup (chunk, row): the sum of the chunk's weights.
__global__ __launch_bounds__(256) void prob_sums_kernel(ProbArgs a) {
    __shared__ __attribute__((aligned(16))) Exp2 e;
    __shared__ unsigned long long red[4];
    const uint32_t r = blockIdx.y, v0 = blockIdx.x * kProbChunk;
    exp2_load(a.exp2, e);
    const int64_t top = (int64_t)(a.keys[r] >> 18) - ((int64_t)1 << 45);
    __syncthreads();
    const int64_t* s = a.scores + (size_t)r * a.lds;
    const uint32_t c = a.inverse[r];
    unsigned long long sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kProbChunk / 256; i++) {
        const uint32_t v = v0 + 256 * i + threadIdx.x;
        if (v < a.vocab) sum += weight(e, top - s[v], c);
    }
    sum = block_sum64(sum, red);
    if (threadIdx.x == 0) {
        a.part[r * kProbChunksMax + blockIdx.x] = sum;
        if (blockIdx.x == 0) a.top[r] = top;
    }
}

// The sum of row r's weights, by one wavefront (uniform over it).
__device__ __forceinline__ uint64_t row_total(const ProbArgs& a, uint32_t r, uint32_t chunks) {
    const uint32_t lane = threadIdx.x & 63;
    unsigned long long z = 0;
    for (uint32_t i = lane; i < chunks; i += 64) z += a.part[r * kProbChunksMax + i];
    return wave_sum64(z);
}

// Workgroup (chunk, row): the chunk's probabilities.
__global__ __launch_bounds__(256) void probs_kernel(ProbArgs a, uint32_t* probs) {
    __shared__ __attribute__((aligned(16))) Exp2 e;
    const uint32_t r = blockIdx.y, v0 = blockIdx.x * kProbChunk;
    exp2_load(a.exp2, e);
    const uint64_t z = row_total(a, r, gridDim.x);
    const double inv = 1.0 / (double)z;
    const int64_t top = a.top[r];
    __syncthreads();
    const int64_t* s = a.scores + (size_t)r * a.lds;
    const uint32_t c = a.inverse[r];
    uint32_t* out = probs + (size_t)r * a.vocab;
#pragma unroll
    for (uint32_t i = 0; i < kProbChunk / 256; i++) {
        const uint32_t v = v0 + 256 * i + threadIdx.x;
        if (v < a.vocab) out[v] = prob32(weight(e, top - s[v], c), z, inv);
    }
    // the keys are 0 between calls; nothing of this launch reads them
    if (blockIdx.x == 0 && r == 0 && threadIdx.x < 8) a.keys[threadIdx.x] = 0;
}

// Workgroup (chunk, request): the request's drafts tested, then the chunk's
// part of the distribution its next token is drawn from; the request's last
// workgroup draws it.
__global__ __launch_bounds__(256) void verify_kernel(VerifyArgs a) {
    __shared__ __attribute__((aligned(16))) Exp2 e;
    __shared__ unsigned long long red[4];
    __shared__ uint64_t total[8];
    __shared__ uint32_t pdraft[8], taken[8], lds_last;
    __shared__ unsigned long long before;
    __shared__ uint32_t chunk;
    const uint32_t tid = threadIdx.x, wave = tid >> 6, chunks = gridDim.x;
    const uint32_t j = blockIdx.y, first = a.first[j], count = a.count[j];
    exp2_load(a.p.exp2, e);
    for (uint32_t i = wave; i <= count; i += 4) {
        const uint64_t z = row_total(a.p, first + i, chunks);
        if ((tid & 63) == 0) total[i] = z;
    }
    __syncthreads();
    auto prob = [&](uint32_t i, uint32_t v) {  // P of the request's row i
        const uint32_t r = first + i;
        const uint64_t z = total[i];
        return prob32(weight(e, a.p.top[r] - a.p.scores[(size_t)r * a.p.lds + v], a.p.inverse[r]),
                      z, 1.0 / (double)z);
    };
    auto drafted = [&](uint32_t i, uint32_t v) -> uint32_t {  // Q
        if (a.q) return a.q[(size_t)(a.draft0[j] + i) * a.p.vocab + v];
        return v == a.draft[first + i] ? 0xffffffffu : 0u;
    };
    if (tid < count) {
        const uint32_t x = a.draft[first + tid], p = prob(tid, x);
        pdraft[tid] = p;
        taken[tid] = (uint64_t)a.accept_u[first + tid] * drafted(tid, x) < (uint64_t)p << 32;
    }
    __syncthreads();
    uint32_t at = 0;
    while (at < count && taken[at]) at++;
    // what is left of P where a token is drawn
    auto above = [&](uint32_t p, uint32_t v) -> uint32_t {
        if (at == count) return p;
        const uint32_t q = drafted(at, v);
        return p > q ? p - q : 0;
    };
    const uint32_t v0 = blockIdx.x * kProbChunk;
    unsigned long long sl = 0, sp = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < kProbChunk / 256; i++) {
        const uint32_t v = v0 + 256 * i + tid;
        if (v < a.p.vocab) {
            const uint32_t p = prob(at, v);
            sl += above(p, v);
            sp += p;
        }
    }
    sl = block_sum64(sl, red);
    sp = block_sum64(sp, red);
    unsigned long long* left = a.left + (size_t)j * kProbChunksMax * 2;
    if (tid == 0) {
        st_coherent(&left[2 * blockIdx.x], sl);
        st_coherent(&left[2 * blockIdx.x + 1], sp);
    }
    if (!arrive_last(a.count_in + 32 * j, chunks, &lds_last)) return;

    // ---- the draw ----
    unsigned long long cl = 0, cp = 0;
    if (tid < chunks) {
        cl = ld_coherent(&left[2 * tid]);
        cp = ld_coherent(&left[2 * tid + 1]);
    }
    const unsigned long long all_l = block_sum64(cl, red), all_p = block_sum64(cp, red);
    const bool whole = all_l == 0;  // nothing above Q: P itself
    const uint64_t sum = whole ? all_p : all_l;  // 1 .. 2^32
    const uint64_t t = ((uint64_t)a.sample_u[j] * sum) >> 32;
    // the chunk, then the thread's scores of it, whose running sum passes t:
    // one thread of the workgroup each time
    const unsigned long long mass_c = whole ? cp : cl;
    const unsigned long long below_c = block_below64(mass_c, red);
    if (t >= below_c && t < below_c + mass_c) {
        chunk = tid;
        before = below_c;
    }
    __syncthreads();
    const uint32_t ch = chunk;
    // the chunk's scores, 8 in a row per thread
    constexpr uint32_t kEach = kProbChunk / 256;
    uint32_t mass[kEach], pv[kEach];
    unsigned long long mine = 0;
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) {
        const uint32_t v = ch * kProbChunk + kEach * tid + i;
        mass[i] = pv[i] = 0;
        if (v < a.p.vocab) {
            pv[i] = prob(at, v);
            mass[i] = whole ? pv[i] : above(pv[i], v);
        }
        mine += mass[i];
    }
    uint64_t lower = before + block_below64(mine, red);
    if (t >= lower && t < lower + mine) {
        uint32_t i = 0;
        while (lower + mass[i] <= t) lower += mass[i++];
        a.host[j] = at;
        a.host[8 + j] = ch * kProbChunk + kEach * tid + i;
        a.host[16 + first + count] = pv[i];
    }
    if (tid < count) a.host[16 + first + tid] = pdraft[tid];
    // the request's words, then its arrival, reach the host before the flag
    __threadfence_system();
    __syncthreads();
    if (tid != 0) return;
    const uint32_t done = __hip_atomic_fetch_add(a.count_in + 32 * 8, 1u, __ATOMIC_ACQ_REL,
                                                 __HIP_MEMORY_SCOPE_AGENT);
    if (done != a.requests - 1) return;
    __hip_atomic_store(a.count_in + 32 * 8, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (uint32_t r = 0; r < 8; r++) a.p.keys[r] = 0;  // nothing of this launch reads them
    __hip_atomic_store(a.flag, a.seq, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_SYSTEM);
}

uint32_t chunks_of(const ProbArgs& a) { return (a.vocab + kProbChunk - 1) / kProbChunk; }

}  // namespace

hipError_t launch_probs(const ProbArgs& a, uint32_t* probs, hipStream_t st) {
    const dim3 grid(chunks_of(a), a.rows);
    prob_sums_kernel<<<grid, 256, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    probs_kernel<<<grid, 256, 0, st>>>(a, probs);
    return hipGetLastError();
}

hipError_t launch_verify(const VerifyArgs& a, hipStream_t st) {
    prob_sums_kernel<<<dim3(chunks_of(a.p), a.p.rows), 256, 0, st>>>(a.p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    verify_kernel<<<dim3(chunks_of(a.p), a.requests), 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace llm
