// shared_attention.hip -- attention of a batch whose sequences share a
// prefix: its K / V once in the context's pages, each sequence's continuation
// in rows of its own.
//
// Every row's values are those of the prompt attention (op 17) over its
// concatenated positions: tiles of 64 from position 0 on, per tile the scores
// s, the running maximum m, p = e14(s - m), the tile's values, and the
// recurrence
//   sum = sat32(rnd(sum old, 16) + sum p),  old = e14(m before - m)
//   acc = sat32(sat32(rnd(acc old, 16)) + value),  out = rnd(acc / sum).
// The recurrence rounds at each tile and so stays a chain over the tiles; all
// that feeds it does not, once the running maxima are known.  Three launches:
//   scores   per (KV head, tile): K converted once to byte planes for the
//            matrix cores and multiplied with every query row of the batch;
//            scores and their maxima to memory;
//   values   per (KV head, tile): each row's running maximum from the maxima
//            of the tiles before, p from it, p V on the matrix cores;
//   join     per (row, head elements): the chain over the tiles.
// A prefix tile is one job for all sequences (16 query rows per product: the
// heads of a KV group of several sequences side by side), so its K / V pass
// through the chip once, not once per sequence; a sequence's own tiles are
// jobs of its own, the first of them beginning with the prefix's last
// positions where the prefix ends inside a tile.
#include "shared_attention.h"

#include "attn_common.h"
#include "mfma_common.h"

namespace llm {
namespace {

__device__ __forceinline__ s16x2 halves(uint32_t w) { return __builtin_bit_cast(s16x2, w); }
__device__ __forceinline__ uint32_t word(s16x2 v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ uint32_t add128(uint32_t w) {
    const s16x2 c = {128, 128};
    return word(halves(w) + c);
}
__device__ __forceinline__ uint32_t max_halves(uint32_t a, uint32_t b) {
    return word(__builtin_elementwise_max(halves(a), halves(b)));
}
// Two values saturated to 16 bits in one word (v_cvt_pk_i16_i32).
__device__ __forceinline__ uint32_t sat_pack(int32_t lo, int32_t hi) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pk_i16(lo, hi));
}
// A group of 8 values in natural order from the bank-paired one (words (0 4)
// (1 5) (2 6) (3 7)).
__device__ __forceinline__ v4u unpair8(v4u n) {
    v4u r;
    r.x = __builtin_amdgcn_perm(n.y, n.x, 0x05040100u);
    r.y = __builtin_amdgcn_perm(n.w, n.z, 0x05040100u);
    r.z = __builtin_amdgcn_perm(n.y, n.x, 0x07060302u);
    r.w = __builtin_amdgcn_perm(n.w, n.z, 0x07060302u);
    return r;
}
__device__ __forceinline__ uint32_t low_plane(uint32_t w0, uint32_t w1) {
    return __builtin_amdgcn_perm(w1, w0, 0x06040200u);
}
// Byte planes (a, b) of 16 values clamped to [-2048, 2048]; `even` and `odd`
// collect the halves' maxima over the words' banks (0 1) and (2 3).
__device__ __forceinline__ void planes16(v4u lo, v4u hi, v4i& a, v4i& b, uint32_t& even,
                                         uint32_t& odd) {
    const uint32_t w[8] = {clamp_word(lo.x), clamp_word(lo.y), clamp_word(lo.z),
                           clamp_word(lo.w), clamp_word(hi.x), clamp_word(hi.y),
                           clamp_word(hi.z), clamp_word(hi.w)};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        even = max_halves(even, w[2 * i]);
        odd = max_halves(odd, w[2 * i + 1]);
        a[i] = (int32_t)plane_c(add128(w[2 * i]), add128(w[2 * i + 1]));
        b[i] = (int32_t)low_plane(w[2 * i], w[2 * i + 1]);
    }
}
// c(x) of both halves, as signed-split planes' words.
__device__ __forceinline__ uint32_t corr_word(uint32_t w) {
    return pack16(sat_corr((int16_t)(w & 0xffffu)), sat_corr((int32_t)w >> 16));
}
__device__ __forceinline__ void corr_planes16(v4u x, v4u y, v4i& h, v4i& l) {
    const uint32_t c[8] = {corr_word(x.x), corr_word(x.y), corr_word(x.z), corr_word(x.w),
                           corr_word(y.x), corr_word(y.y), corr_word(y.z), corr_word(y.w)};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        h[i] = (int32_t)plane_c(add128(c[2 * i]), add128(c[2 * i + 1]));
        l[i] = (int32_t)low_plane(c[2 * i], c[2 * i + 1]);
    }
}

constexpr uint32_t kJobPieces = 4, kJobRows = 16 * kJobPieces;

// What a workgroup works on: a tile of one KV head and rows [rho, end), in
// pieces of 16 from rho on.
struct Job {
    uint32_t h, j;          // KV head, tile
    uint32_t rho, end;
    uint32_t seq;           // own tiles: the sequence
    uint32_t base, valid;   // first position, positions of the tile that count
    bool own;
};
__device__ __forceinline__ uint32_t length_of(const SharedAttnArgs& a, uint32_t seq) {
    const uint32_t n = a.own_cap ? a.own_len[seq] : 0;
    return n < a.own_cap ? n : a.own_cap;
}
__device__ __forceinline__ bool job_of(const SharedAttnArgs& a, Job& b) {
    b.own = blockIdx.x >= a.shared_jobs;
    if (!b.own) {
        const uint32_t grp = blockIdx.x % a.groups, tile = blockIdx.x / a.groups;
        b.h = tile / a.whole;
        b.j = tile % a.whole;
        b.rho = kJobRows * grp;
        b.end = min(b.rho + kJobRows, a.rows);
        b.seq = 0;
        b.base = 64 * b.j;
        b.valid = 64;
        return true;
    }
    const uint32_t id = blockIdx.x - a.shared_jobs;
    const uint32_t o = id % a.own_tiles, th = id / a.own_tiles;
    b.h = th % a.kv_heads;
    b.seq = th / a.kv_heads;
    b.j = a.whole + o;
    b.rho = b.seq * a.group;
    b.end = b.rho + a.group;
    b.base = 64 * b.j;
    const uint32_t n = a.prefix + length_of(a, b.seq);
    if (b.base >= n) return false;
    b.valid = min(n - b.base, 64u);
    return true;
}

// The K row of position `pos` of the job's tile (in pages: bank-paired), or
// null where there is none.
__device__ __forceinline__ const int16_t* k_row(const SharedAttnArgs& a, const Job& b,
                                                uint32_t pos, bool& in_page) {
    in_page = !b.own || pos < a.prefix;
    if (in_page)
        return a.kcache + ((size_t)b.h * a.pages + b.j) * TILE * a.head_dim +
               (pos & 63) * a.head_dim;
    if (pos >= b.base + b.valid) return nullptr;
    return a.k_own + ((size_t)b.seq * a.kv_heads + b.h) * a.own_cap * a.head_dim +
           (size_t)(pos - a.prefix) * a.head_dim;
}
// Elements of row rho's query in front of it in q (at most 64 x 2,048).
__device__ __forceinline__ uint32_t q_at(const SharedAttnArgs& a, uint32_t h, uint32_t rho) {
    const uint32_t seq = __umul24(rho, a.inv_group) >> 16;  // rho / group
    return (rho + __umul24(seq, (a.kv_heads - 1) * a.group) + h * a.group) * a.head_dim;
}

// The score by the definition: four banks of AP_RND-narrowed products, each
// saturating as its products arrive.
__device__ __noinline__ int32_t defined_score(const int16_t* q, const int16_t* k, bool in_page,
                                              uint32_t d, int32_t qk_scale) {
    int32_t bank[4] = {0, 0, 0, 0};
    for (uint32_t e = 0; e < d; e += 4) {
#pragma unroll
        for (uint32_t u = 0; u < 4; u++) {
            const int32_t kv = k[in_page ? paired(e + u) : e + u];
            const int32_t t = (int32_t)fx_rnd((int64_t)q[e + u] * fx_fm_to_wt(kv), 4);
            bank[u] = fx_sat32((int64_t)bank[u] + t);
        }
    }
    int32_t t = fx_sat32((int64_t)bank[0] + bank[1] + bank[2] + bank[3]);
    t = fx_sat32(fx_rnd((int64_t)t * ((int64_t)qk_scale << 8), 16));
    return fx_sat16(fx_rnd(t, 8));
}

// Scores of the job's rows: wavefront w the tile's positions 16 w .. + 15, so
// that each K value is loaded and converted once per workgroup, and the byte
// planes of piece w's queries for all of them.  KC: 64-element chunks of a
// head.
template <int KC>
struct ScoreSmem {
    int8_t q[kJobPieces][KC][2][1024];  // c, d
    int8_t corr[kJobPieces][KC][2][1024];  // c(q), where a key value saturates
    int32_t max[kJobRows][4];
    uint32_t far;
};
template <int KC, bool OWN>
__device__ __forceinline__ void score_job(const SharedAttnArgs& a, const Job& b,
                                          ScoreSmem<KC>& sm) {
    const uint32_t lane = threadIdx.x & 63, q = lane & 15, g = lane >> 4, d = a.head_dim;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t nrows = b.end - b.rho;
    const v4i zero = {0, 0, 0, 0};
    const v4u none = {0, 0, 0, 0};
    bool in_page;
    const int16_t* row = k_row(a, b, b.base + 16 * w + q, in_page);
    v4u raw[KC][2], qx[KC], qy[KC];
#pragma unroll
    for (int kc = 0; kc < KC; kc++) {
        const uint32_t e = 64 * kc + 16 * g;
        raw[kc][0] = raw[kc][1] = none;
        if (e < d && (!OWN || row)) {
            raw[kc][0] = *(const v4u*)(row + e);
            raw[kc][1] = *(const v4u*)(row + e + 8);
        }
    }
    const bool piece = 16 * w < nrows;  // the wavefront has one
    if (piece) {
        // rows past the last repeat it
        const int16_t* qr = a.q + q_at(a, b.h, b.rho + min(16 * w + q, nrows - 1));
#pragma unroll
        for (int kc = 0; kc < KC; kc++) {
            const uint32_t e = 64 * kc + 16 * g;
            qx[kc] = qy[kc] = none;
            if (e < d) {
                qx[kc] = *(const v4u*)(qr + e);
                qy[kc] = *(const v4u*)(qr + e + 8);
            }
        }
    }
    if (threadIdx.x == 0) sm.far = 0;
    v4i ka[KC], kb[KC], bias;
    uint32_t even = 0x80008000u, odd = 0x80008000u;
    {
        const v4i ones = {0x01010101, 0x01010101, 0x01010101, 0x01010101};
        v4i sa = zero, sb = zero;
#pragma unroll
        for (int kc = 0; kc < KC; kc++) {
            v4u x = raw[kc][0], y = raw[kc][1];
            if (!OWN || in_page) x = unpair8(x), y = unpair8(y);
            planes16(x, y, ka[kc], kb[kc], even, odd);
            sa = mfma16(ka[kc], ones, sa);
            sb = mfma16(kb[kc], ones, sb);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) bias[i] = 128 * (256 * sa[i] + sb[i]);
    }
    if (piece) {
#pragma unroll
        for (int kc = 0; kc < KC; kc++) {
            const v4u u = qx[kc], v = qy[kc];
            *(v4i*)&sm.q[w][kc][0][16 * lane] =
                v4i{(int32_t)plane_c(u.x, u.y), (int32_t)plane_c(u.z, u.w),
                    (int32_t)plane_c(v.x, v.y), (int32_t)plane_c(v.z, v.w)};
            *(v4i*)&sm.q[w][kc][1][16 * lane] =
                v4i{(int32_t)plane_d(u.x, u.y), (int32_t)plane_d(u.z, u.w),
                    (int32_t)plane_d(v.x, v.y), (int32_t)plane_d(v.z, v.w)};
        }
    }
    // a key value saturates; a lane's part of a bank is all -2048, without
    // which no bank passes 2^31 - 1 (32 products of -32768 and -2048)
    const bool far = __any(sat_mask(max_halves(even, odd)) != 0);
    constexpr uint32_t kLow = 0xf800f800u;
    const uint32_t le = even ^ kLow, lo = odd ^ kLow;
    const bool low = KC == 2 && __any((le & 0xffffu) == 0 || (le >> 16) == 0 ||
                                      (lo & 0xffffu) == 0 || (lo >> 16) == 0);
    __syncthreads();
    if (far) sm.far = 1;
    __syncthreads();
    const bool kf = sm.far != 0;
    if (kf) {
        if (piece) {
#pragma unroll
            for (int kc = 0; kc < KC; kc++) {
                v4i qh, ql;
                corr_planes16(qx[kc], qy[kc], qh, ql);
                *(v4i*)&sm.corr[w][kc][0][16 * lane] = qh;
                *(v4i*)&sm.corr[w][kc][1][16 * lane] = ql;
            }
        }
        __syncthreads();
    }
    int16_t* out = a.scores +
                   (((size_t)b.h * a.tiles + b.j) * a.rows_pad + b.rho) * TILE + 16 * w + 4 * g;
#pragma unroll 1
    for (uint32_t r0 = 0; r0 < nrows; r0 += 16) {
        const uint32_t p = r0 / 16;
        v4i ac = zero, x = zero, bd = bias;
#pragma unroll
        for (int kc = 0; kc < KC; kc++) {
            const v4i qc = *(const v4i*)&sm.q[p][kc][0][16 * lane];
            const v4i qd = *(const v4i*)&sm.q[p][kc][1][16 * lane];
            ac = mfma16(ka[kc], qc, ac);
            x = mfma16(ka[kc], qd, x);
            bd = mfma16(kb[kc], qd, bd);
            x = mfma16(kb[kc], qc, x);
        }
        if (kf) {
#pragma unroll
            for (int kc = 0; kc < KC; kc++) {
                const v4i mk = mask2048(ka[kc], kb[kc]);
                x = mfma16(mk, *(const v4i*)&sm.corr[p][kc][0][16 * lane], x);
                bd = mfma16(mk, *(const v4i*)&sm.corr[p][kc][1][16 * lane], bd);
            }
        }
        int32_t sc[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            // sum = 256 t + lo; the two roundings of sum * scale are
            // floor((sum qk + 2^7 + 2^15) / 2^16) in one, and a t past 2^23 (a
            // sum past 32 bits) saturates the score
            const int32_t t = (ac[i] << 8) + x[i] + (bd[i] >> 8);
            const int32_t lw = __mul24(bd[i] & 255, a.qk_scale) + 32896;
            sc[i] = (__mul24(med3(t, -(1 << 23), (1 << 23) - 1), a.qk_scale) + (lw >> 8)) >> 8;
        }
        if (low) {
            const int16_t* qr = a.q + q_at(a, b.h, b.rho + min(r0 + q, nrows - 1));
#pragma unroll 1
            for (int i = 0; i < 4; i++) {
                bool paged;
                const int16_t* kr = k_row(a, b, b.base + 16 * w + 4 * g + i, paged);
                if (!OWN || kr) {
                    const int32_t v = defined_score(qr, kr, paged, d, a.qk_scale);
                    sc[0] = i == 0 ? v : sc[0];
                    sc[1] = i == 1 ? v : sc[1];
                    sc[2] = i == 2 ? v : sc[2];
                    sc[3] = i == 3 ? v : sc[3];
                }
            }
        }
        if (OWN) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (16 * w + 4 * g + i >= b.valid) sc[i] = INT16_MIN;
        }
        const uint32_t s0 = sat_pack(sc[0], sc[1]), s1 = sat_pack(sc[2], sc[3]);
        const uint32_t m = max_halves(s0, s1);
        const int32_t mx = quad_max(max((int32_t)(int16_t)(m & 0xffffu), (int32_t)m >> 16));
        if (r0 + q < nrows) {
            *(v2u*)(out + (r0 + q) * TILE) = v2u{s0, s1};
            if (g == 0) sm.max[r0 + q][w] = mx;
        }
    }
    __syncthreads();
    const uint32_t r = threadIdx.x;
    if (r < nrows) {
        const v4i m = *(const v4i*)sm.max[r];
        a.tmax[((size_t)b.h * a.tiles + b.j) * a.rows_pad + b.rho + r] =
            (int16_t)max(max(m[0], m[1]), max(m[2], m[3]));
    }
}

template <int KC>
__global__ __launch_bounds__(256, 4) void shared_scores_kernel(SharedAttnArgs a) {
    __shared__ __attribute__((aligned(16))) ScoreSmem<KC> sm;
    Job b;
    if (!job_of(a, b)) return;
    if (b.own)
        score_job<KC, true>(a, b, sm);
    else
        score_job<KC, false>(a, b, sm);
}

// LDS row of a head element of an own tile: 64 positions, and 16 bytes so that
// rows start in different banks.
constexpr uint32_t kOwnRow = 72;

// The own tile's V rows into `vt` [d][kOwnRow], positions in natural order.
__device__ __forceinline__ void own_values(const SharedAttnArgs& a, const Job& b, int16_t* vt) {
    const uint32_t tid = threadIdx.x, d = a.head_dim;
    // positions of the tile that lie in the prefix: its last page's
    const uint32_t head = b.base < a.prefix ? a.prefix - b.base : 0;  // < 64
    const int16_t* page = a.vcache + ((size_t)b.h * a.pages + b.j) * TILE * d;
    const int16_t* own = a.v_own + ((size_t)b.seq * a.kv_heads + b.h) * a.own_cap * d;
    // positions p and p + 1, 8 elements at a time
    const uint32_t e = 8 * (tid & 15);
    if (e >= d) return;
#pragma unroll
    for (uint32_t i = 0; i < 2; i++) {
        const uint32_t p = 2 * (tid >> 4) + 32 * i;
        v4u x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
        if (p >= head && p < b.valid)
            x = *(const v4u*)(own + (size_t)(b.base + p - a.prefix) * d + e);
        if (p + 1 >= head && p + 1 < b.valid)
            y = *(const v4u*)(own + (size_t)(b.base + p + 1 - a.prefix) * d + e);
        if (p < head) {
#pragma unroll
            for (int u = 0; u < 4; u++)
                x[u] = pack16(page[(e + 2 * u) * TILE + paired(p)],
                              page[(e + 2 * u + 1) * TILE + paired(p)]);
        }
        if (p + 1 < head) {
#pragma unroll
            for (int u = 0; u < 4; u++)
                y[u] = pack16(page[(e + 2 * u) * TILE + paired(p + 1)],
                              page[(e + 2 * u + 1) * TILE + paired(p + 1)]);
        }
        int16_t* o = vt + e * kOwnRow + p;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            *(uint32_t*)(o + (2 * u) * kOwnRow) = __builtin_amdgcn_perm(y[u], x[u], 0x05040100u);
            *(uint32_t*)(o + (2 * u + 1) * kOwnRow) =
                __builtin_amdgcn_perm(y[u], x[u], 0x07060302u);
        }
    }
}

struct ValueSmem {
    int16_t e14[2056];
    int16_t hist[4][kJobRows];   // per wavefront, running maximum of its tiles
    uint32_t far;                // a V value saturates
    uint32_t pad[3];
    int8_t planes[kJobPieces][4][1024];  // p, c(p); own tiles use the first
    int16_t vt[128 * kOwnRow];   // own tiles
};
typedef short s16x8 __attribute__((ext_vector_type(8)));

// Values of the job's rows: wavefront w forms the probabilities of piece w's
// rows, and the values of 16-element strips w, w + 4 for all of them.  ES:
// strips per wavefront.
template <int ES, bool OWN>
__device__ __forceinline__ void value_job(const SharedAttnArgs& a, const Job& b, ValueSmem& sm) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, q = lane & 15, g = lane >> 4;
    const uint32_t w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t d = a.head_dim, ne = d / 16, nrows = b.end - b.rho;
    // this tile's rows from b.rho on
    const size_t trow = ((size_t)b.h * a.tiles + b.j) * a.rows_pad + b.rho;
    v4u raw[ES][2];
    if (!OWN) {
        const int16_t* page = a.vcache + ((size_t)b.h * a.pages + b.j) * TILE * d;
#pragma unroll
        for (int es = 0; es < ES; es++) {
            const uint32_t e = 16 * min(w + 4 * es, ne - 1) + q;  // past the last: repeated
            raw[es][0] = *(const v4u*)(page + e * TILE + 16 * g);
            raw[es][1] = *(const v4u*)(page + e * TILE + 16 * g + 8);
        }
    }
    v4u table = {0, 0, 0, 0}, last = {0, 0, 0, 0};
    table = *(const v4u*)(a.exp14 + 8 * tid);
    if (tid == 0) last = *(const v4u*)(a.exp14 + 2048);
    // the lane's row of piece w (rows past the last repeat it): positions 16 g
    // .. + 15 and the tile's maximum
    const bool piece = 16 * w < nrows;
    const uint32_t r = min(16 * w + q, nrows - 1);
    v4u s0 = {0, 0, 0, 0}, s1 = s0;
    int32_t tmj = 0;
    if (piece) {
        s0 = *(const v4u*)(a.scores + trow * TILE + r * TILE + 16 * g);
        s1 = *(const v4u*)(a.scores + trow * TILE + r * TILE + 16 * g + 8);
        tmj = a.tmax[trow + r];
    }
    // the running maxima before this tile: threads over (8 rows, every 32nd tile)
    const uint32_t r8 = b.rho & ~7u, skip = b.rho - r8, grp = tid & 7;
    s16x8 m = (short)INT16_MIN;
    if (r8 + 8 * grp < b.end) {
        const int16_t* tm = a.tmax + (size_t)b.h * a.tiles * a.rows_pad + r8 + 8 * grp;
#pragma unroll 4
        for (uint32_t t = tid >> 3; t < b.j; t += 32)
            m = __builtin_elementwise_max(m, *(const s16x8*)(tm + (size_t)t * a.rows_pad));
    }
    if (OWN) own_values(a, b, sm.vt);
    *(v4u*)(sm.e14 + 8 * tid) = table;
    if (tid == 0) {
        *(v4u*)(sm.e14 + 2048) = last;
        sm.far = 0;
    }
    // over the wavefront's lanes of equal tid % 8, then through LDS
    {
        v4u x = __builtin_bit_cast(v4u, m);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t v = x[i];
            v = max_halves(v, (uint32_t)__builtin_amdgcn_update_dpp(
                                  0, (int32_t)v, 0x128, 0xf, 0xf, false));  // row_ror:8
            const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
            v = max_halves(s[0], s[1]);
            const auto t = __builtin_amdgcn_permlane32_swap(v, v, false, false);
            x[i] = max_halves(t[0], t[1]);
        }
        if (lane < 8) *(v4u*)&sm.hist[w][8 * lane] = x;
    }
    __syncthreads();
    // ---- probabilities, as operand planes ----
    uint32_t pw[8];
    if (piece) {
        int32_t before = INT16_MIN;
#pragma unroll
        for (int u = 0; u < 4; u++) before = max(before, (int32_t)sm.hist[u][skip + r]);
        const int32_t top = max(before, tmj);
        const uint32_t tops = pack16(top, top);
        const s16x2 floor2 = {-2048, -2048};
        int32_t sum = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // sat16(s - top), not below -2048
            const uint32_t s = i < 4 ? s0[i] : s1[i - 4];
            const s16x2 x = __builtin_elementwise_max(
                __builtin_elementwise_sub_sat(halves(s), halves(tops)), floor2);
            int32_t p0 = sm.e14[x.x + 2048], p1 = sm.e14[x.y + 2048];
            if (OWN) {
                p0 = 16 * g + 2 * i < b.valid ? p0 : 0;
                p1 = 16 * g + 2 * i + 1 < b.valid ? p1 : 0;
            }
            pw[i] = pack16(p0, p1);
            sum = dot2(pw[i], 0x00010001u, sum);
        }
        v4i pc, pd;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            // p + 128 <= 16512: no carry between the halves
            pc[i] = (int32_t)plane_c(pw[2 * i] + 0x00800080u, pw[2 * i + 1] + 0x00800080u);
            pd[i] = (int32_t)low_plane(pw[2 * i], pw[2 * i + 1]);
        }
        *(v4i*)&sm.planes[w][0][16 * lane] = pc;
        *(v4i*)&sm.planes[w][1][16 * lane] = pd;
        sum = quad_sum(sum);
        if (g == 0 && 16 * w + q < nrows) {
            a.tsum[trow + r] = sum << 2;
            a.old[trow + r] = (int32_t)sm.e14[max(before - top, -2048) + 2048] << 2;
        }
    }
    v4i va[ES], vb[ES];
    uint32_t even = 0x80008000u, odd = 0x80008000u;
#pragma unroll
    for (int es = 0; es < ES; es++) {
        if (OWN) {
            const uint32_t e = 16 * min(w + 4 * es, ne - 1) + q;
            const int16_t* p = sm.vt + e * kOwnRow + 16 * g;
            planes16(*(const v4u*)p, *(const v4u*)(p + 8), va[es], vb[es], even, odd);
        } else {
            planes16(unpair8(raw[es][0]), unpair8(raw[es][1]), va[es], vb[es], even, odd);
        }
    }
    if (__any(sat_mask(max_halves(even, odd)) != 0)) sm.far = 1;
    __syncthreads();
    const bool vf = sm.far != 0;
    if (vf) {
        if (piece) {
            v4i ph, pq;
            corr_planes16(v4u{pw[0], pw[1], pw[2], pw[3]}, v4u{pw[4], pw[5], pw[6], pw[7]}, ph, pq);
            *(v4i*)&sm.planes[w][2][16 * lane] = ph;
            *(v4i*)&sm.planes[w][3][16 * lane] = pq;
        }
        __syncthreads();
    }
    // ---- values ----
    const v4i zero = {0, 0, 0, 0}, half = {8224, 8224, 8224, 8224};
    int16_t* out = a.tval + trow * d + 4 * g;
#pragma unroll 1
    for (uint32_t r0 = 0; r0 < nrows; r0 += 16) {
        const int8_t(*pl)[1024] = sm.planes[r0 / 16];
        const v4i pc = *(const v4i*)&pl[0][lane * 16], pd = *(const v4i*)&pl[1][lane * 16];
        v4i ph = zero, pq = zero;
        if (vf) {
            ph = *(const v4i*)&pl[2][lane * 16];
            pq = *(const v4i*)&pl[3][lane * 16];
        }
        const bool real = r0 + q < nrows;
#pragma unroll
        for (int es = 0; es < ES; es++) {
            v4i ac = mfma16(va[es], pc, zero);
            v4i x = mfma16(va[es], pd, zero);
            v4i bd = mfma16(vb[es], pd, half);
            x = mfma16(vb[es], pc, x);
            if (vf) {
                const v4i mk = mask2048(va[es], vb[es]);
                x = mfma16(mk, ph, x);
                bd = mfma16(mk, pq, bd);
            }
            int32_t tv[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                // sums in [-2^31, 2^31 - 2^16] (64 products of at most 2^14
                // and -2048, or 2048 with its correction of -1024): exact in
                // 32 bits, and so with 8224 added; rnd(rnd(tot, 6), 8) =
                // floor((tot + 2^5 + 2^13) / 2^14)
                const uint32_t tot = ((((uint32_t)ac[i] << 8) + (uint32_t)x[i]) << 8) +
                                     (uint32_t)bd[i];
                tv[i] = (int32_t)tot >> 14;
            }
            const uint32_t st = w + 4 * es;
            if (real && st < ne)
                *(v2u*)(out + (r0 + q) * d + 16 * st) =
                    v2u{sat_pack(tv[0], tv[1]), sat_pack(tv[2], tv[3])};
        }
    }
}

template <int ES>
__global__ __launch_bounds__(256, 4) void shared_values_kernel(SharedAttnArgs a) {
    __shared__ __attribute__((aligned(16))) ValueSmem sm;
    Job b;
    if (!job_of(a, b)) return;
    if (b.own)
        value_job<ES, true>(a, b, sm);
    else
        value_job<ES, false>(a, b, sm);
}

// The chain over a row's tiles, one workgroup per row and 64 head elements.  A
// thread loads 8 of the elements of 8 consecutive tiles (a run), all of them at once, and leaves
// them and their sums over the run in LDS; a wavefront then walks the runs
// while the next block's loads are under way.  A run over which the maximum does not
// rise (old = 1.0 throughout: most, once the first tiles are past) is one
// addition of its sum, four such runs at a time: exact, because the
// probabilities' sums are not negative and the elements' 32 values (at most
// 2^28 together) cannot saturate an accumulator within 2^30.
__global__ __launch_bounds__(256) void shared_join_kernel(SharedAttnArgs a) {
    constexpr uint32_t EC = 8, RUNS = 256 / EC, BLOCK = 8 * RUNS;
    __shared__ __attribute__((aligned(16))) int16_t s_v[BLOCK][8 * EC];
    __shared__ __attribute__((aligned(16))) int32_t s_run[RUNS][8 * EC];
    __shared__ __attribute__((aligned(16))) int32_t s_old[BLOCK], s_sum[BLOCK];
    __shared__ __attribute__((aligned(16))) int32_t s_all[RUNS][2];  // same, sum
    const uint32_t tid = threadIdx.x, ec = tid % EC, run = tid / EC;
    const uint32_t h = blockIdx.x / a.rows, rho = blockIdx.x % a.rows;
    const uint32_t d = a.head_dim, e0 = 8 * EC * blockIdx.y, ne = min(d - e0, 8 * EC);
    const uint32_t seq = __umul24(rho, a.inv_group) >> 16;
    const size_t at = (size_t)h * a.tiles * a.rows_pad + rho;
    const uint32_t step = a.rows_pad;
    const bool real = 8 * ec < ne;
    v4u v[8];
    int32_t old = 65536, ts = 0;
    // (bounded by the tiles there can be: nothing waits for the length)
    auto load = [&](uint32_t t0) {
        const uint32_t first = t0 + 8 * run;
        const int16_t* src = a.tval + (at + (size_t)first * step) * d + e0 + 8 * ec;
#pragma unroll
        for (uint32_t u = 0; u < 8; u++) {
            v[u] = v4u{0, 0, 0, 0};
            if (real && first + u < a.tiles) v[u] = *(const v4u*)(src + (size_t)u * step * d);
        }
        if (tid < BLOCK && t0 + tid < a.tiles) {
            old = a.old[at + (size_t)(t0 + tid) * step];
            ts = a.tsum[at + (size_t)(t0 + tid) * step];
        }
    };
    load(0);
    const uint32_t n = a.prefix + length_of(a, seq), nt = (n + 63) / 64;
    int32_t sum = 0, acc = 0;
#pragma unroll 1
    for (uint32_t t0 = 0; t0 < nt; t0 += BLOCK) {
        const uint32_t first = t0 + 8 * run;
        int32_t lo[4] = {0, 0, 0, 0}, hi[4] = {0, 0, 0, 0};
#pragma unroll
        for (uint32_t u = 0; u < 8; u++) {
            // tiles that this sequence does not have hold anything
            if (first + u >= nt) v[u] = v4u{0, 0, 0, 0};
            *(v4u*)&s_v[8 * run + u][8 * ec] = v[u];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                lo[i] = dot2(v[u][i], 0x00000001u, lo[i]);
                hi[i] = dot2(v[u][i], 0x00010000u, hi[i]);
            }
        }
        *(v4i*)&s_run[run][8 * ec] = v4i{lo[0], hi[0], lo[1], hi[1]};
        *(v4i*)&s_run[run][8 * ec + 4] = v4i{lo[2], hi[2], lo[3], hi[3]};
        if (tid < BLOCK) {
            const bool there = t0 + tid < nt;
            int32_t o = there ? old : 65536, z = there ? ts : 0;
            s_old[tid] = o;
            s_sum[tid] = z;
            // over the 8 tiles of a run: quad_perm [1 0 3 2], [2 3 0 1], row_half_mirror
            o &= dpp<0xb1, 0xf>(o, o);
            o &= dpp<0x4e, 0xf>(o, o);
            o &= dpp<0x141, 0xf>(o, o);
            z += dpp<0xb1, 0xf>(z, z);
            z += dpp<0x4e, 0xf>(z, z);
            z += dpp<0x141, 0xf>(z, z);
            if (tid % 8 == 0) {
                s_all[tid / 8][0] = o;  // old <= 2^16, and that only without a rise
                s_all[tid / 8][1] = z;
            }
        }
        if (t0 + BLOCK < nt) load(t0 + BLOCK);
        lds_barrier();
        if (tid < ne) {
            // four runs at a time; those past the last tile add nothing
            const uint32_t runs = min((nt - t0 + 7) / 8, RUNS);
#pragma unroll 1
            for (uint32_t r = 0; r < runs; r += 4) {
                const v4i a0 = *(const v4i*)s_all[r], a1 = *(const v4i*)s_all[r + 2];
                int32_t whole[4];
#pragma unroll
                for (int u = 0; u < 4; u++) whole[u] = s_run[r + u][tid];
                const bool near = __all(((uint32_t)acc + (1u << 30)) >> 31 == 0);
                if ((a0[0] & a0[2] & a1[0] & a1[2]) == 65536 && near) {
                    acc += (whole[0] + whole[1] + whole[2] + whole[3]) << 8;
                    sum = __builtin_elementwise_add_sat(sum, a0[1] + a0[3] + a1[1] + a1[3]);
                    continue;
                }
#pragma unroll 1
                for (uint32_t t = 8 * r; t < 8 * r + 32; t += 8) {
                    if (s_all[t / 8][0] == 65536 && near) {
                        acc += s_run[t / 8][tid] << 8;
                        sum = __builtin_elementwise_add_sat(sum, s_all[t / 8][1]);
                        continue;
                    }
                    const v4i o0 = *(const v4i*)&s_old[t], o1 = *(const v4i*)&s_old[t + 4];
                    const v4i z0 = *(const v4i*)&s_sum[t], z1 = *(const v4i*)&s_sum[t + 4];
                    int32_t x[8];
#pragma unroll
                    for (int u = 0; u < 8; u++) x[u] = (int32_t)s_v[t + u][tid] << 8;
#pragma unroll
                    for (int u = 0; u < 8; u++) {
                        const int32_t o = u < 4 ? o0[u] : o1[u - 4], z = u < 4 ? z0[u] : z1[u - 4];
                        sum = __builtin_elementwise_add_sat(rnd16_mul(sum, o), z);
                        acc = __builtin_elementwise_add_sat(rnd16_mul(acc, o), x[u]);
                    }
                }
            }
        }
        lds_barrier();
    }
    if (tid < ne) {
        const int32_t inv = fx_inv_sum(sum);
        a.out[q_at(a, h, rho) + e0 + tid] = sat16_32(rnd16_mul(acc, inv));
    }
}

uint32_t round_to(uint32_t v, uint32_t m) { return (v + m - 1) / m * m; }
size_t part_bytes(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

void shared_attention_shape(SharedAttnArgs& a) {
    a.whole = a.prefix / 64;
    const uint32_t tail = a.prefix % 64 + a.own_cap;
    a.own_tiles = (tail + 63) / 64;
    a.tiles = a.whole + a.own_tiles;
    a.rows = a.sequences * a.group;
    a.rows_pad = round_to(a.rows, 16);
    a.inv_group = (65536 + a.group - 1) / a.group;  // rho < 1,024, group <= 16: exact
    a.groups = (a.rows + kJobRows - 1) / kJobRows;
    a.shared_jobs = a.kv_heads * a.whole * a.groups;
    a.own_jobs = a.kv_heads * a.sequences * a.own_tiles;
}

size_t shared_attention_bytes(const SharedAttnArgs& a) {
    const size_t rt = (size_t)a.kv_heads * a.tiles * a.rows_pad;
    return part_bytes(rt * 64 * 2) + part_bytes(rt * 2) + 2 * part_bytes(rt * 4) +
           part_bytes(rt * a.head_dim * 2);
}

void shared_attention_scratch(SharedAttnArgs& a, uint8_t* base) {
    const size_t rt = (size_t)a.kv_heads * a.tiles * a.rows_pad;
    auto take = [&](size_t bytes) {
        uint8_t* p = base;
        base += part_bytes(bytes);
        return p;
    };
    a.scores = (int16_t*)take(rt * 64 * 2);
    a.tmax = (int16_t*)take(rt * 2);
    a.old = (int32_t*)take(rt * 4);
    a.tsum = (int32_t*)take(rt * 4);
    a.tval = (int16_t*)take(rt * a.head_dim * 2);
}

hipError_t launch_shared_attention(const SharedAttnArgs& a, hipStream_t st) {
    const uint32_t grid = a.shared_jobs + a.own_jobs;
    if (grid) {
        if (a.head_dim <= 64)
            shared_scores_kernel<1><<<grid, 256, 0, st>>>(a);
        else
            shared_scores_kernel<2><<<grid, 256, 0, st>>>(a);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        if (a.head_dim <= 64)
            shared_values_kernel<1><<<grid, 256, 0, st>>>(a);
        else
            shared_values_kernel<2><<<grid, 256, 0, st>>>(a);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    const dim3 rows(a.kv_heads * a.rows, (a.head_dim + 63) / 64);
    shared_join_kernel<<<rows, 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace llm
