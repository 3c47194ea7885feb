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
// scores' pass reads it once, one row in 100 us, 6.2 TB/s, and writes 8 bytes
// per score, 8 rows in 110); what follows are two short passes over the scores,
// a workgroup per chunk of them and row (or request): the weights' sums, a
// request's last workgroup to arrive testing its drafts, then the
// probabilities, or the draws, a request's last workgroup drawing its token.
// Dependent round trips bound those (arrivals, the chunks' sums, the chunk
// again, the words to the host, ~1 us each), not the scores' bytes: sums of 8
// rows 10.3 us at 151,936 tokens, 7.5 at 32,011; draws 11.4 and 11.1; both in
// one launch, 4 rows of 1,024, 11.0; probabilities of 8 rows 4.7 at 32,011.
#include "verify.h"

#include "attn_common.h"
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

// Sum over the wavefront's lanes up to this one: within rows of 16 lanes, then
// the row before's and the first half's (row_bcast).
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long scan_step64(unsigned long long v) {
    const uint32_t lo = (uint32_t)dpp<CTRL, ROWS>(0, (int32_t)v);
    const uint32_t hi = (uint32_t)dpp<CTRL, ROWS>(0, (int32_t)(v >> 32));
    return v + ((unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ unsigned long long wave_scan64(unsigned long long v) {
    v = scan_step64<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
    v = scan_step64<0x112, 0xf>(v);
    v = scan_step64<0x114, 0xf>(v);
    v = scan_step64<0x118, 0xf>(v);
    v = scan_step64<0x142, 0xa>(v);  // row_bcast:15, 31
    return scan_step64<0x143, 0xc>(v);
}
// Over all of them, uniform.
__device__ __forceinline__ unsigned long long wave_sum64(unsigned long long v) {
    v = wave_scan64(v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int32_t)v, 63);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int32_t)(v >> 32), 63);
    return (unsigned long long)hi << 32 | lo;
}
// Sums over the workgroup's 256 threads, uniform; red: 8 words.
__device__ __forceinline__ void block_sums64(unsigned long long& u, unsigned long long& v,
                                             unsigned long long* red) {
    u = wave_sum64(u);
    v = wave_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        red[threadIdx.x >> 6] = u;
        red[4 + (threadIdx.x >> 6)] = v;
    }
    __syncthreads();
    u = red[0] + red[1] + red[2] + red[3];
    v = red[4] + red[5] + red[6] + red[7];
}

// Sum of v over the threads below this one; red: 4 words.
__device__ __forceinline__ unsigned long long block_below64(unsigned long long v,
                                                            unsigned long long* red) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned long long s = wave_scan64(v);
    __syncthreads();
    if (lane == 63) red[wave] = s;
    __syncthreads();
    for (uint32_t w = 0; w < wave; w++) s += red[w];
    return s - v;
}

// Q of a request's draft row i at token v.
__device__ __forceinline__ uint32_t drafted(const ProbArgs& a, uint32_t j, uint32_t i,
                                            uint32_t v) {
    if (a.q) return a.q[(size_t)(a.draft0[j] + i) * a.vocab + v];
    return v == a.draft[a.first[j] + i] ? 0xffffffffu : 0u;
}

// The chunk's part of the distribution that request j's next token is drawn
// from (row `at` of it, whose weights' sum and largest score are z and top);
// the request's last workgroup of `chunks` draws it.  The tables are in e.
struct DrawSmem {
    unsigned long long red[8], before;
    uint32_t last, chunk;
};
__device__ __forceinline__ void draw_chunk(const ProbArgs& a, const Exp2& e, DrawSmem& sm,
                                           uint32_t own, uint32_t chunks, uint32_t j, uint32_t at,
                                           uint64_t z, int64_t top, const uint32_t* pdraft) {
    const uint32_t tid = threadIdx.x, first = a.first[j], count = a.count[j], row = first + at;
    const double inv = 1.0 / (double)z;
    const uint32_t c = a.inverse[row];
    constexpr uint32_t kEach = kProbChunk / 256;
    // P of the thread's tokens of a chunk, and what of it lies above Q (`at`
    // past the drafts: all of it)
    uint32_t p[kEach], above[kEach];
    auto fill = [&](uint32_t ch) {
        const uint32_t v = ch * kProbChunk + kEach * tid;
        int64_t sv[kEach];
        uint32_t q[kEach];
#pragma unroll
        for (uint32_t i = 0; i < kEach; i++) {
            const uint32_t t = v + i;
            sv[i] = a.scores[score_at(t < a.vocab ? t : 0, row, a.rows)];
            q[i] = at < count && t < a.vocab ? drafted(a, j, at, t) : 0;
        }
        __syncthreads();  // (the tables, the first time)
#pragma unroll
        for (uint32_t i = 0; i < kEach; i++) {
            p[i] = 0;
            if (v + i < a.vocab) p[i] = prob32(weight(e, top - sv[i], c), z, inv);
            above[i] = p[i] > q[i] ? p[i] - q[i] : 0;
        }
    };
    fill(own);
    unsigned long long sl = 0, sp = 0;
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) sl += above[i], sp += p[i];
    block_sums64(sl, sp, sm.red);
    if (chunks > 1) {
        unsigned long long* left = a.left + (size_t)j * kProbChunksMax * 2;
        if (tid == 0) {
            st_coherent(&left[2 * own], sl);
            st_coherent(&left[2 * own + 1], sp);
        }
        if (!arrive_last(a.count_in + 32 * j, chunks, &sm.last)) return;
        sl = sp = 0;
        if (tid < chunks) {
            sl = ld_coherent(&left[2 * tid]);
            sp = ld_coherent(&left[2 * tid + 1]);
        }
    } else if (tid != 0) {
        sl = sp = 0;
    }
    unsigned long long all_l = sl, all_p = sp;
    block_sums64(all_l, all_p, sm.red);
    const bool whole = all_l == 0;  // nothing above Q: P itself
    const uint64_t sum = whole ? all_p : all_l;  // 1 .. 2^32
    const uint64_t t = ((uint64_t)a.sample_u[j] * sum) >> 32;
    // the chunk, then the thread's tokens of it, whose running sum passes t:
    // one thread of the workgroup each time
    const unsigned long long mass_c = whole ? sp : sl;
    const unsigned long long below_c = block_below64(mass_c, sm.red);
    if (t >= below_c && t < below_c + mass_c) {
        sm.chunk = tid;
        sm.before = below_c;
    }
    __syncthreads();
    const uint32_t ch = sm.chunk;
    if (ch != own) fill(ch);
    unsigned long long mine = 0;
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) {
        if (whole) above[i] = p[i];
        mine += above[i];
    }
    auto tell = [&](uint32_t i, uint32_t v) {
        __hip_atomic_store(a.host + i, (unsigned long long)a.seq << 32 | v, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_SYSTEM);
    };
    uint64_t lower = sm.before + block_below64(mine, sm.red);
    if (t >= lower && t < lower + mine) {
        uint32_t at_i = 0, pv = p[0];
#pragma unroll
        for (uint32_t i = 0; i + 1 < kEach; i++)
            if (at_i == i && lower + above[i] <= t) {
                lower += above[i];
                at_i = i + 1;
                pv = p[i + 1];
            }
        tell(j, at);
        tell(8 + j, ch * kProbChunk + kEach * tid + at_i);
        tell(16 + first + count, pv);
    }
    if (tid < count) tell(16 + first + tid, pdraft[tid]);
    if (tid <= count) a.keys[first + tid] = 0;  // nothing of this launch reads them
}

// Workgroup (chunk, row): the sum of the chunk's weights.  The last one of a
// request tests its drafts and, where a chunk of draws holds the vocabulary
// (DRAW), draws its token too.
template <bool DRAW>
__global__ __launch_bounds__(256) void prob_sums_kernel(ProbArgs a) {
    __shared__ __attribute__((aligned(16))) Exp2 e;
    __shared__ DrawSmem sm;
    __shared__ unsigned long long total[8];
    __shared__ uint32_t pdraft[8], taken[8], place;
    const uint32_t tid = threadIdx.x, r = blockIdx.y, v0 = blockIdx.x * kSumChunk;
    const uint32_t chunks = gridDim.x, j = a.request[r], first = a.first[j], count = a.count[j];
    constexpr uint32_t kEach = kSumChunk / 256;
    int64_t sv[kEach];
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) {
        const uint32_t v = v0 + 256 * i + tid;
        sv[i] = a.scores[score_at(v < a.vocab ? v : 0, r, a.rows)];
    }
    exp2_load(a.exp2, e);
    const int64_t top = (int64_t)(a.keys[r] >> 18) - ((int64_t)1 << 45);
    __syncthreads();
    const uint32_t c = a.inverse[r];
    unsigned long long sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++)
        if (v0 + 256 * i + tid < a.vocab) sum += weight(e, top - sv[i], c);
    sum = wave_sum64(sum);
    if ((tid & 63) == 0) sm.red[tid >> 6] = sum;
    __syncthreads();
    sum = sm.red[0] + sm.red[1] + sm.red[2] + sm.red[3];
    if (tid == 0) st_coherent(&a.part[r * kSumChunksMax + blockIdx.x], sum);
    // few arrivals on one line (15 ns each), else a row's first (~1 us more)
    if (chunks * (count + 1) <= 64) {
        if (!arrive_last(a.count_in + 32 * (8 + j), chunks * (count + 1), &sm.last)) return;
    } else {
        if (!arrive_last(a.count_in + 32 * r, chunks, &sm.last)) return;
        if (count && !arrive_last(a.count_in + 32 * (8 + j), count + 1, &sm.last)) return;
    }

    // the rows' sums, a wavefront at a time
    for (uint32_t i = tid >> 6; i <= count; i += 4) {
        const uint32_t k = tid & 63;
        const uint64_t z = wave_sum64(
            k < chunks ? ld_coherent(&a.part[(first + i) * kSumChunksMax + k]) : 0);
        if ((tid & 63) == 0) total[i] = z;
    }
    __syncthreads();
    auto row_top = [&](uint32_t i) {
        return (int64_t)(a.keys[first + i] >> 18) - ((int64_t)1 << 45);
    };
    if (tid < count) {
        const uint32_t row = first + tid, x = a.draft[row];
        const uint64_t z = total[tid];
        const int64_t below = row_top(tid) - a.scores[score_at(x, row, a.rows)];
        const uint32_t p = prob32(weight(e, below, a.inverse[row]), z, 1.0 / (double)z);
        pdraft[tid] = p;
        taken[tid] = (uint64_t)a.accept_u[row] * drafted(a, j, tid, x) < (uint64_t)p << 32;
    }
    __syncthreads();
    if (tid == 0) {
        uint32_t at = 0;
        while (at < count && taken[at]) at++;
        place = at;
        if (!DRAW) {
            DrawPlace* o = &a.place[j];
            o->total = total[at];
            o->top = row_top(at);
            o->at = at;
        }
    }
    if constexpr (DRAW) {
        __syncthreads();
        const uint32_t at = place;
        draw_chunk(a, e, sm, 0, 1, j, at, total[at], row_top(at), pdraft);
    } else {
        if (tid < count) a.place[j].pdraft[tid] = pdraft[tid];
    }
}

// Workgroup (chunk, row): the chunk's probabilities.
__global__ __launch_bounds__(256) void probs_kernel(ProbArgs a, uint32_t* probs) {
    __shared__ __attribute__((aligned(16))) Exp2 e;
    const uint32_t tid = threadIdx.x, r = blockIdx.y, v0 = blockIdx.x * kProbChunk;
    int64_t sv[kProbChunk / 256];
#pragma unroll
    for (uint32_t i = 0; i < kProbChunk / 256; i++) {
        const uint32_t v = v0 + 256 * i + tid;
        sv[i] = a.scores[score_at(v < a.vocab ? v : 0, r, a.rows)];
    }
    exp2_load(a.exp2, e);
    const uint64_t z = a.place[r].total;
    const int64_t top = a.place[r].top;
    const double inv = 1.0 / (double)z;
    __syncthreads();
    const uint32_t c = a.inverse[r];
    uint32_t* out = probs + (size_t)r * a.vocab;
#pragma unroll
    for (uint32_t i = 0; i < kProbChunk / 256; i++) {
        const uint32_t v = v0 + 256 * i + tid;
        if (v < a.vocab) out[v] = prob32(weight(e, top - sv[i], c), z, inv);
    }
    // the keys are 0 between calls; nothing of this launch reads them
    if (blockIdx.x == 0 && r == 0 && tid < 8) a.keys[tid] = 0;
}

__global__ __launch_bounds__(256) void draw_kernel(ProbArgs a) {
    __shared__ __attribute__((aligned(16))) Exp2 e;
    __shared__ DrawSmem sm;
    exp2_load(a.exp2, e);
    const DrawPlace& o = a.place[blockIdx.y];
    draw_chunk(a, e, sm, blockIdx.x, gridDim.x, blockIdx.y, o.at, o.total, o.top, o.pdraft);
}

uint32_t chunks_of(const ProbArgs& a, uint32_t each) { return (a.vocab + each - 1) / each; }

}  // namespace

hipError_t launch_probs(const ProbArgs& a, uint32_t* probs, hipStream_t st) {
    prob_sums_kernel<false><<<dim3(chunks_of(a, kSumChunk), a.rows), 256, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    probs_kernel<<<dim3(chunks_of(a, kProbChunk), a.rows), 256, 0, st>>>(a, probs);
    return hipGetLastError();
}

hipError_t launch_verify(const ProbArgs& a, hipStream_t st) {
    // a vocabulary of one chunk: 1,024 tokens 24.1 us a call, 26.3 with the draws
    // in a launch of their own, which larger ones need for their chunks
    if (a.vocab <= kProbChunk) {
        prob_sums_kernel<true><<<dim3(1, a.rows), 256, 0, st>>>(a);
        return hipGetLastError();
    }
    prob_sums_kernel<false><<<dim3(chunks_of(a, kSumChunk), a.rows), 256, 0, st>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    draw_kernel<<<dim3(chunks_of(a, kProbChunk), a.requests), 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace llm
