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
// Measured back to back, 16 query heads in 2 KV groups of 128: 8 sequences,
// 16,000 + up to 300 positions (17.7 MB of K and V, 2.9 us at 6.2 TB/s) 7.0, 9.1
// and 7.7 us, together 25.5; 32 sequences, 8,100 + up to 600: 12.2, 16.7 and
// 9.9, together 39.1.  The first are dependent steps (loads, conversion,
// products, exchange, store) and launch boundaries, not bytes; the second work:
// 1,648 tiles' jobs of 64 rows, and 36 MB of tile values written and read.
// A prefix tile is one job for all sequences (16 query rows per product: the
// heads of a KV group of several sequences side by side), so its K / V pass
// through the chip once, not once per sequence; a sequence's own tiles are
// jobs of its own, the first of them beginning with the prefix's last
// positions where the prefix ends inside a tile.  Up to kSmallTiles tiles, where
// the launches are what takes the time, one launch does all of it.
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

// 16 positions of a tile as operand planes (lane: position lane % 16), their
// bias 128 sum k' as the products' results lie, whether a value saturates, and
// whether a lane's part of a bank is all -2048, without which no bank passes
// 2^31 - 1 (32 products of -32768 and -2048).
template <int KC>
struct KeyPlanes {
    v4i a[KC], b[KC], bias;
    bool far, low;
};
// From raw rows, bank-paired where `paged` (per lane).
template <int KC, bool ANY>
__device__ __forceinline__ void key_planes(const v4u (*raw)[2], bool paged, KeyPlanes<KC>& k) {
    const v4i ones = {0x01010101, 0x01010101, 0x01010101, 0x01010101};
    uint32_t even = 0x80008000u, odd = 0x80008000u;
    v4i sa = {0, 0, 0, 0}, sb = sa;
#pragma unroll
    for (int kc = 0; kc < KC; kc++) {
        v4u x = raw[kc][0], y = raw[kc][1];
        if (!ANY || paged) x = unpair8(x), y = unpair8(y);
        planes16(x, y, k.a[kc], k.b[kc], even, odd);
        sa = mfma16(k.a[kc], ones, sa);
        sb = mfma16(k.b[kc], ones, sb);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) k.bias[i] = 128 * (256 * sa[i] + sb[i]);
    k.far = __any(sat_mask(max_halves(even, odd)) != 0);
    constexpr uint32_t kLow = 0xf800f800u;
    const uint32_t le = even ^ kLow, lo = odd ^ kLow;
    k.low = KC == 2 && __any((le & 0xffffu) == 0 || (le >> 16) == 0 || (lo & 0xffffu) == 0 ||
                             (lo >> 16) == 0);
}
// The raw values of a lane's K row (0 where there is none) or query.
template <int KC>
__device__ __forceinline__ void row_load(const int16_t* row, uint32_t g, uint32_t d,
                                         v4u (*raw)[2]) {
#pragma unroll
    for (int kc = 0; kc < KC; kc++) {
        const uint32_t e = 64 * kc + 16 * g;
        raw[kc][0] = raw[kc][1] = v4u{0, 0, 0, 0};
        if (e < d && row) {
            raw[kc][0] = *(const v4u*)(row + e);
            raw[kc][1] = *(const v4u*)(row + e + 8);
        }
    }
}
// Operand planes in LDS, [KC][2][1024]: c and d of queries, or their c(q).
template <int KC>
__device__ __forceinline__ void query_planes(const v4u (*raw)[2], uint32_t lane,
                                             int8_t (*o)[2][1024]) {
#pragma unroll
    for (int kc = 0; kc < KC; kc++) {
        const v4u u = raw[kc][0], v = raw[kc][1];
        *(v4i*)&o[kc][0][16 * lane] = v4i{(int32_t)plane_c(u.x, u.y), (int32_t)plane_c(u.z, u.w),
                                          (int32_t)plane_c(v.x, v.y), (int32_t)plane_c(v.z, v.w)};
        *(v4i*)&o[kc][1][16 * lane] = v4i{(int32_t)plane_d(u.x, u.y), (int32_t)plane_d(u.z, u.w),
                                          (int32_t)plane_d(v.x, v.y), (int32_t)plane_d(v.z, v.w)};
    }
}
template <int KC>
__device__ __forceinline__ void query_corr(const v4u (*raw)[2], uint32_t lane,
                                           int8_t (*o)[2][1024]) {
#pragma unroll
    for (int kc = 0; kc < KC; kc++) {
        v4i h, l;
        corr_planes16(raw[kc][0], raw[kc][1], h, l);
        *(v4i*)&o[kc][0][16 * lane] = h;
        *(v4i*)&o[kc][1][16 * lane] = l;
    }
}
// Scores of a piece's rows (lane: row lane % 16, query row rho) at positions
// 16 w + 4 g + s of the job's tile, as packed words; positions that do not
// count have the lowest.
template <int KC, bool OWN>
__device__ __forceinline__ v2u piece_scores(const SharedAttnArgs& a, const Job& b,
                                            const KeyPlanes<KC>& k, uint32_t w, uint32_t lane,
                                            uint32_t rho, const int8_t (*qp)[2][1024],
                                            const int8_t (*corr)[2][1024]) {
    const uint32_t g = lane >> 4;
    const v4i zero = {0, 0, 0, 0};
    v4i ac = zero, x = zero, bd = k.bias;
#pragma unroll
    for (int kc = 0; kc < KC; kc++) {
        const v4i qc = *(const v4i*)&qp[kc][0][16 * lane];
        const v4i qd = *(const v4i*)&qp[kc][1][16 * lane];
        ac = mfma16(k.a[kc], qc, ac);
        x = mfma16(k.a[kc], qd, x);
        bd = mfma16(k.b[kc], qd, bd);
        x = mfma16(k.b[kc], qc, x);
    }
    if (k.far) {
#pragma unroll
        for (int kc = 0; kc < KC; kc++) {
            const v4i mk = mask2048(k.a[kc], k.b[kc]);
            x = mfma16(mk, *(const v4i*)&corr[kc][0][16 * lane], x);
            bd = mfma16(mk, *(const v4i*)&corr[kc][1][16 * lane], bd);
        }
    }
    int32_t sc[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        // sum = 256 t + lo; the two roundings of sum * scale are
        // floor((sum qk + 2^7 + 2^15) / 2^16) in one, and a t past 2^23 (a sum
        // past 32 bits) saturates the score
        const int32_t t = (ac[i] << 8) + x[i] + (bd[i] >> 8);
        const int32_t lw = __mul24(bd[i] & 255, a.qk_scale) + 32896;
        sc[i] = (__mul24(med3(t, -(1 << 23), (1 << 23) - 1), a.qk_scale) + (lw >> 8)) >> 8;
    }
    if (k.low) {
        const int16_t* qr = a.q + q_at(a, b.h, rho);
#pragma unroll 1
        for (int i = 0; i < 4; i++) {
            bool paged;
            const int16_t* kr = k_row(a, b, b.base + 16 * w + 4 * g + i, paged);
            if (!OWN || kr) {
                const int32_t v = defined_score(qr, kr, paged, a.head_dim, a.qk_scale);
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
    return v2u{sat_pack(sc[0], sc[1]), sat_pack(sc[2], sc[3])};
}
// The largest of a row's scores over the lanes that hold it.
__device__ __forceinline__ int32_t row_max(v2u s) {
    const uint32_t m = max_halves(s.x, s.y);
    return quad_max(max((int32_t)(int16_t)(m & 0xffffu), (int32_t)m >> 16));
}

// Scores of the job's rows: wavefront w the tile's positions 16 w .. + 15, so
// that each K value is loaded and converted once per workgroup, and the byte
// planes of piece w's queries for all of them.  KC: 64-element chunks of a
// head.
template <int KC>
struct ScoreSmem {
    int8_t q[kJobPieces][KC][2][1024];
    int8_t corr[kJobPieces][KC][2][1024];  // where a key value saturates
    int32_t max[kJobRows][4];
    uint32_t far;
};
template <int KC, bool OWN>
__device__ __forceinline__ void score_job(const SharedAttnArgs& a, const Job& b,
                                          ScoreSmem<KC>& sm) {
    const uint32_t lane = threadIdx.x & 63, q = lane & 15, g = lane >> 4, d = a.head_dim;
    const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t nrows = b.end - b.rho;
    bool paged;
    v4u kraw[KC][2], qraw[KC][2];
    row_load<KC>(k_row(a, b, b.base + 16 * w + q, paged), g, d, kraw);
    const bool piece = 16 * w < nrows;  // the wavefront has one
    if (piece)  // rows past the last repeat it
        row_load<KC>(a.q + q_at(a, b.h, b.rho + min(16 * w + q, nrows - 1)), g, d, qraw);
    if (threadIdx.x == 0) sm.far = 0;
    KeyPlanes<KC> k;
    key_planes<KC, OWN>(kraw, paged, k);
    if (piece) query_planes<KC>(qraw, lane, sm.q[w]);
    __syncthreads();
    if (k.far) sm.far = 1;
    __syncthreads();
    if (sm.far != 0) {
        if (piece) query_corr<KC>(qraw, lane, sm.corr[w]);
        __syncthreads();
    }
    int16_t* out = a.scores +
                   (((size_t)b.h * a.tiles + b.j) * a.rows_pad + b.rho) * TILE + 16 * w + 4 * g;
#pragma unroll 1
    for (uint32_t r0 = 0; r0 < nrows; r0 += 16) {
        const uint32_t p = r0 / 16;
        const v2u s = piece_scores<KC, OWN>(a, b, k, w, lane, b.rho + min(r0 + q, nrows - 1),
                                            sm.q[p], sm.corr[p]);
        const int32_t mx = row_max(s);
        if (r0 + q < nrows) {
            *(v2u*)(out + (r0 + q) * TILE) = s;
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

// Probabilities of a lane's 16 positions (natural order) from their scores and
// the running maximum, as packed words, and their sum; MASK: positions from
// `valid` on, counted from the lane's first, have none.
template <bool MASK>
__device__ __forceinline__ int32_t row_probs(v4u s0, v4u s1, int32_t top, int32_t valid,
                                             const int16_t* e14, uint32_t* pw) {
    const uint32_t tops = pack16(top, top);
    const s16x2 floor2 = {-2048, -2048};
    int32_t sum = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        // sat16(s - top), not below -2048
        const uint32_t s = i < 4 ? s0[i] : s1[i - 4];
        const s16x2 x = __builtin_elementwise_max(
            __builtin_elementwise_sub_sat(halves(s), halves(tops)), floor2);
        int32_t p0 = e14[x.x + 2048], p1 = e14[x.y + 2048];
        if (MASK) {
            p0 = 2 * i < valid ? p0 : 0;
            p1 = 2 * i + 1 < valid ? p1 : 0;
        }
        pw[i] = pack16(p0, p1);
        sum = dot2(pw[i], 0x00010001u, sum);
    }
    return sum;
}
// Their operand planes in LDS, [4][1024]: p, and (corr) c(p).
__device__ __forceinline__ void prob_planes(const uint32_t* pw, uint32_t lane,
                                            int8_t (*o)[1024]) {
    v4i pc, pd;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        // p + 128 <= 16512: no carry between the halves
        pc[i] = (int32_t)plane_c(pw[2 * i] + 0x00800080u, pw[2 * i + 1] + 0x00800080u);
        pd[i] = (int32_t)low_plane(pw[2 * i], pw[2 * i + 1]);
    }
    *(v4i*)&o[0][16 * lane] = pc;
    *(v4i*)&o[1][16 * lane] = pd;
}
__device__ __forceinline__ void prob_corr(const uint32_t* pw, uint32_t lane, int8_t (*o)[1024]) {
    v4i ph, pq;
    corr_planes16(v4u{pw[0], pw[1], pw[2], pw[3]}, v4u{pw[4], pw[5], pw[6], pw[7]}, ph, pq);
    *(v4i*)&o[2][16 * lane] = ph;
    *(v4i*)&o[3][16 * lane] = pq;
}
// Tile values of a strip (lane: row lane % 16, elements 4 (lane / 16) + s) as
// packed words.
__device__ __forceinline__ v2u strip_values(v4i va, v4i vb, bool far, uint32_t lane,
                                            const int8_t (*pl)[1024]) {
    const v4i zero = {0, 0, 0, 0}, half = {8224, 8224, 8224, 8224};
    const v4i pc = *(const v4i*)&pl[0][16 * lane], pd = *(const v4i*)&pl[1][16 * lane];
    v4i ac = mfma16(va, pc, zero);
    v4i x = mfma16(va, pd, zero);
    v4i bd = mfma16(vb, pd, half);
    x = mfma16(vb, pc, x);
    if (far) {
        const v4i mk = mask2048(va, vb);
        x = mfma16(mk, *(const v4i*)&pl[2][16 * lane], x);
        bd = mfma16(mk, *(const v4i*)&pl[3][16 * lane], bd);
    }
    int32_t tv[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        // sums in [-2^31, 2^31 - 2^16] (64 products of at most 2^14 and -2048,
        // or 2048 with its correction of -1024): exact in 32 bits, and so with
        // 8224 added; rnd(rnd(tot, 6), 8) = floor((tot + 2^5 + 2^13) / 2^14)
        const uint32_t tot = ((((uint32_t)ac[i] << 8) + (uint32_t)x[i]) << 8) + (uint32_t)bd[i];
        tv[i] = (int32_t)tot >> 14;
    }
    return v2u{sat_pack(tv[0], tv[1]), sat_pack(tv[2], tv[3])};
}

struct ValueSmem {
    int16_t e14[2056];
    int16_t hist[4][kJobRows];   // per wavefront, running maximum of its tiles
    uint32_t far;                // a V value saturates
    uint32_t pad[3];
    union {
        int8_t planes[kJobPieces][4][1024];  // p, c(p) of the pieces
        struct {                             // own tiles have one
            int8_t planes[4][1024];
            int16_t vt[128 * kOwnRow];
        } own;
    };
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
    auto planes_of = [&](uint32_t piece) { return OWN ? sm.own.planes : sm.planes[piece]; };
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
    if (OWN) own_values(a, b, sm.own.vt);
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
        const int32_t sum = quad_sum(row_probs<OWN>(
            s0, s1, top, (int32_t)b.valid - 16 * (int32_t)g, sm.e14, pw));
        prob_planes(pw, lane, planes_of(w));
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
            const int16_t* p = sm.own.vt + e * kOwnRow + 16 * g;
            planes16(*(const v4u*)p, *(const v4u*)(p + 8), va[es], vb[es], even, odd);
        } else {
            planes16(unpair8(raw[es][0]), unpair8(raw[es][1]), va[es], vb[es], even, odd);
        }
    }
    if (__any(sat_mask(max_halves(even, odd)) != 0)) sm.far = 1;
    __syncthreads();
    const bool vf = sm.far != 0;
    if (vf) {
        if (piece) prob_corr(pw, lane, planes_of(w));
        __syncthreads();
    }
    // ---- values ----
    int16_t* out = a.tval + trow * d + 4 * g;
#pragma unroll 1
    for (uint32_t r0 = 0; r0 < nrows; r0 += 16) {
        const bool real = r0 + q < nrows;
#pragma unroll
        for (int es = 0; es < ES; es++) {
            const v2u tv = strip_values(va[es], vb[es], vf, lane, planes_of(r0 / 16));
            const uint32_t st = w + 4 * es;
            if (real && st < ne) *(v2u*)(out + (r0 + q) * d + 16 * st) = tv;
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
// thread loads 8 of the elements of 8 consecutive tiles (a run), all of them
// at once, and leaves them and their sums over the run in LDS; a wavefront then
// walks the runs while the next block's loads are under way.  A run over which
// the maximum does not rise (old = 1.0 throughout: most, once the first tiles
// are past) is one addition of its sum, four such runs at a time: exact,
// because the probabilities' sums are not negative and the elements' 32 values
// (at most 2^28 together) cannot saturate an accumulator within 2^30.
// RUNS: of a block, by as many groups of 8 threads.
template <uint32_t RUNS>
__global__ __launch_bounds__(256) void shared_join_kernel(SharedAttnArgs a) {
    constexpr uint32_t EC = 8, BLOCK = 8 * RUNS;
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
    const bool mine = run < RUNS, real = mine && 8 * ec < ne;
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
            if (mine) *(v4u*)&s_v[8 * run + u][8 * ec] = v[u];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                lo[i] = dot2(v[u][i], 0x00000001u, lo[i]);
                hi[i] = dot2(v[u][i], 0x00010000u, hi[i]);
            }
        }
        if (mine) {
            *(v4i*)&s_run[run][8 * ec] = v4i{lo[0], hi[0], lo[1], hi[1]};
            *(v4i*)&s_run[run][8 * ec + 4] = v4i{lo[2], hi[2], lo[3], hi[3]};
        }
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

// Few tiles: the whole attention of one sequence and KV head by one workgroup:
// scores (wavefront w positions 16 w .. + 15 of each tile), probabilities
// (wavefront w tile w's), values and the chain (wavefront w strips w, w + 4,
// the accumulators in registers).  One launch in place of three, but the shared
// tiles' keys and values are converted for each sequence, and a workgroup takes
// its tiles one after another.  Back to back, this and the three launches: head
// dimension 64, 2 KV heads, 8 sequences: 2 tiles 7.9 and 12.5 us, 4 tiles 10.2
// and 12.5, 8 tiles 16.1 and 12.6; dimension 128: 2 tiles 10.9 and 14.6, 4
// tiles 14.8 and 15.4, 8 tiles 24.1 and 15.6.  8 KV heads, 64 sequences, 4
// tiles: 20.4 and 39.0.
constexpr uint32_t kSmallTiles = 4;
template <int KC>
struct SmallSmem {
    int8_t q[KC][2][1024], corr[KC][2][1024];
    int16_t e14[2056];
    int16_t s[kSmallTiles][16][72];      // scores; rows 144 bytes apart
    int32_t max[kSmallTiles][16][4];
    int32_t old[kSmallTiles][16], sum[kSmallTiles][16];
    int8_t planes[kSmallTiles][4][1024];
    int16_t vt[128 * kOwnRow];
};
template <int KC>
__global__ __launch_bounds__(256) void shared_small_kernel(SharedAttnArgs a) {
    constexpr int ES = KC;
    __shared__ __attribute__((aligned(16))) SmallSmem<KC> sm;
    const uint32_t tid = threadIdx.x, lane = tid & 63, q = lane & 15, g = lane >> 4;
    const uint32_t w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t d = a.head_dim, ne = d / 16;
    Job b;
    b.h = blockIdx.x % a.kv_heads;
    b.seq = blockIdx.x / a.kv_heads;
    b.rho = b.seq * a.group;
    b.end = b.rho + a.group;
    b.own = true;
    const uint32_t rho = min(b.rho + q, b.end - 1);  // rows past the last repeat it
    if (w == 0) {
        v4u qraw[KC][2];
        row_load<KC>(a.q + q_at(a, b.h, rho), g, d, qraw);
        query_planes<KC>(qraw, lane, sm.q);
        query_corr<KC>(qraw, lane, sm.corr);
    }
    *(v4u*)(sm.e14 + 8 * tid) = *(const v4u*)(a.exp14 + 8 * tid);
    if (tid == 0) *(v4u*)(sm.e14 + 2048) = *(const v4u*)(a.exp14 + 2048);
    const uint32_t n = a.prefix + length_of(a, b.seq), nt = (n + 63) / 64;
    int32_t before = INT16_MIN, total = 0, acc[ES][4];
#pragma unroll
    for (int es = 0; es < ES; es++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[es][i] = 0;
    if (nt > 0) {  // the whole workgroup alike
        auto tile = [&](uint32_t t) {
            b.j = t;
            b.base = 64 * t;
            b.valid = min(n - b.base, 64u);
        };
        v4u kraw[kSmallTiles][KC][2];
        bool paged[kSmallTiles];
#pragma unroll
        for (uint32_t i = 0; i < kSmallTiles; i++) {
            tile(min(i, nt - 1));
            row_load<KC>(k_row(a, b, b.base + 16 * w + q, paged[i]), g, d, kraw[i]);
        }
        __syncthreads();  // the queries' planes
#pragma unroll
        for (uint32_t i = 0; i < kSmallTiles; i++) {
            if (i >= nt) break;
            tile(i);
            KeyPlanes<KC> k;
            key_planes<KC, true>(kraw[i], paged[i], k);
            const v2u s = piece_scores<KC, true>(a, b, k, w, lane, rho, sm.q, sm.corr);
            *(v2u*)&sm.s[i][q][16 * w + 4 * g] = s;
            const int32_t mx = row_max(s);
            if (g == 0) sm.max[i][q][w] = mx;
        }
        __syncthreads();
        // ---- probabilities ----
#pragma unroll
        for (uint32_t i = 0; i < kSmallTiles; i++) {
            if (i >= nt) break;
            const v4i m = *(const v4i*)sm.max[i][q];
            const int32_t next = max(before, max(max(m[0], m[1]), max(m[2], m[3])));
            if (i == w) {
                tile(i);
                uint32_t pw[8];
                const int32_t sum = quad_sum(row_probs<true>(
                    *(const v4u*)&sm.s[i][q][16 * g], *(const v4u*)&sm.s[i][q][16 * g + 8], next,
                    (int32_t)b.valid - 16 * (int32_t)g, sm.e14, pw));
                prob_planes(pw, lane, sm.planes[i]);
                prob_corr(pw, lane, sm.planes[i]);
                if (g == 0) {
                    sm.sum[i][q] = sum << 2;
                    sm.old[i][q] = (int32_t)sm.e14[max(before - next, -2048) + 2048] << 2;
                }
            }
            before = next;
        }
        // ---- values and the chain ----
#pragma unroll 1
        for (uint32_t i = 0; i < nt; i++) {
            tile(i);
            const bool page = b.base + 64 <= a.prefix;  // all of it in one
            if (!page) {
                if (i > 0) __syncthreads();  // what the last tile's strips read
                own_values(a, b, sm.vt);
            }
            if (!page || i == 0) __syncthreads();
            const int32_t old = sm.old[i][q];
            total = __builtin_elementwise_add_sat(rnd16_mul(total, old), sm.sum[i][q]);
            const int16_t* src = a.vcache + ((size_t)b.h * a.pages + b.j) * TILE * d;
#pragma unroll
            for (int es = 0; es < ES; es++) {
                const uint32_t e = 16 * min(w + 4 * es, ne - 1) + q;  // past the last: repeated
                v4u x, y;
                if (page) {
                    x = unpair8(*(const v4u*)(src + e * TILE + 16 * g));
                    y = unpair8(*(const v4u*)(src + e * TILE + 16 * g + 8));
                } else {
                    x = *(const v4u*)(sm.vt + e * kOwnRow + 16 * g);
                    y = *(const v4u*)(sm.vt + e * kOwnRow + 16 * g + 8);
                }
                v4i va, vb;
                uint32_t even = 0x80008000u, odd = 0x80008000u;
                planes16(x, y, va, vb, even, odd);
                const v2u tv = strip_values(va, vb, __any(sat_mask(max_halves(even, odd)) != 0),
                                            lane, sm.planes[i]);
#pragma unroll
                for (int u = 0; u < 4; u++)
                    acc[es][u] = __builtin_elementwise_add_sat(rnd16_mul(acc[es][u], old),
                                                               half16(tv, u) << 8);
            }
        }
    }
    const int32_t inv = fx_inv_sum(total);
    int16_t* out = a.out + q_at(a, b.h, rho) + 4 * g;
#pragma unroll
    for (int es = 0; es < ES; es++) {
        int32_t y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) y[i] = rnd16_mul(acc[es][i], inv);
        if (q < a.group && w + 4 * es < ne)
            *(v2u*)(out + 16 * (w + 4 * es)) = v2u{sat_pack(y[0], y[1]), sat_pack(y[2], y[3])};
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
    if (a.tiles <= kSmallTiles) return 0;
    const size_t rt = (size_t)a.kv_heads * a.tiles * a.rows_pad;
    return part_bytes(rt * 64 * 2) + part_bytes(rt * 2) + 2 * part_bytes(rt * 4) +
           part_bytes(rt * a.head_dim * 2);
}

void shared_attention_scratch(SharedAttnArgs& a, uint8_t* base) {
    if (a.tiles <= kSmallTiles) return;
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
    if (a.tiles <= kSmallTiles) {
        const uint32_t grid = a.kv_heads * a.sequences;
        if (a.head_dim <= 64)
            shared_small_kernel<1><<<grid, 256, 0, st>>>(a);
        else
            shared_small_kernel<2><<<grid, 256, 0, st>>>(a);
        return hipGetLastError();
    }
    const uint32_t grid = a.shared_jobs + a.own_jobs;
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
    const dim3 rows(a.kv_heads * a.rows, (a.head_dim + 63) / 64);
    // 32 runs take 43 KB of LDS (3 workgroups per compute unit), 28 take 38 (4):
    // the larger blocks where all rows' workgroups run at once all the same (255
    // tiles: 7.7 us and 8.9), the smaller where they do not (1,024 workgroups,
    // 136 tiles: 12.2 and 9.9)
    if (rows.x * rows.y > 3 * 256)
        shared_join_kernel<28><<<rows, 256, 0, st>>>(a);
    else
        shared_join_kernel<32><<<rows, 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace llm
