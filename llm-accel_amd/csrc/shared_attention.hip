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

__device__ __forceinline__ uint32_t add128(uint32_t w) {
    const s16x2 c = {128, 128};
    return __builtin_bit_cast(uint32_t, (s16x2)(__builtin_bit_cast(s16x2, w) + c));
}
// Words (0 4) (1 5) (2 6) (3 7) of a group of 8 values in natural order.
__device__ __forceinline__ v4u pair8(v4u n) {
    v4u r;
    r.x = __builtin_amdgcn_perm(n.z, n.x, 0x05040100u);
    r.y = __builtin_amdgcn_perm(n.z, n.x, 0x07060302u);
    r.z = __builtin_amdgcn_perm(n.w, n.y, 0x05040100u);
    r.w = __builtin_amdgcn_perm(n.w, n.y, 0x07060302u);
    return r;
}
__device__ __forceinline__ uint32_t low_plane(uint32_t w0, uint32_t w1) {
    return __builtin_amdgcn_perm(w1, w0, 0x06040200u);
}
// Byte planes (a, b) of 16 clamped values; `any` collects saturating ones.
__device__ __forceinline__ void planes16(v4u lo, v4u hi, v4i& a, v4i& b, uint32_t& any) {
    const v4u x = clamp4(lo, any), y = clamp4(hi, any);
    a[0] = (int32_t)plane_c(add128(x.x), add128(x.y));
    a[1] = (int32_t)plane_c(add128(x.z), add128(x.w));
    a[2] = (int32_t)plane_c(add128(y.x), add128(y.y));
    a[3] = (int32_t)plane_c(add128(y.z), add128(y.w));
    b[0] = (int32_t)low_plane(x.x, x.y);
    b[1] = (int32_t)low_plane(x.z, x.w);
    b[2] = (int32_t)low_plane(y.x, y.y);
    b[3] = (int32_t)low_plane(y.z, y.w);
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

// What a wavefront works on: a tile of one KV head and row pieces of 16.
struct Job {
    uint32_t h, j;          // KV head, tile
    uint32_t rho, end;      // rows [rho, end), in pieces of 16
    uint32_t seq;           // own tiles: the sequence
    uint32_t base, valid;   // first position, positions of the tile that count
    bool own;
};
__device__ __forceinline__ uint32_t length_of(const SharedAttnArgs& a, uint32_t seq) {
    const uint32_t n = a.own_cap ? a.own_len[seq] : 0;
    return n < a.own_cap ? n : a.own_cap;
}
__device__ __forceinline__ bool job_of(const SharedAttnArgs& a, uint32_t shared_blocks, Job& b) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    b.own = blockIdx.x >= shared_blocks;
    if (!b.own) {
        const uint32_t id = blockIdx.x * 4 + wave;
        if (id >= a.shared_jobs) return false;
        const uint32_t grp = id % a.groups, tile = id / a.groups;
        b.h = tile / a.whole;
        b.j = tile % a.whole;
        b.rho = 16 * a.per_wave * grp;
        b.end = min(b.rho + 16 * a.per_wave, a.rows);
        b.seq = 0;
        b.base = 64 * b.j;
        b.valid = 64;
        return true;
    }
    const uint32_t id = (blockIdx.x - shared_blocks) * 4 + wave;
    if (id >= a.own_jobs) return false;
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
                                                uint32_t pos, bool& paired_order) {
    paired_order = true;
    if (!b.own || pos < a.prefix)
        return a.kcache + (((size_t)b.h * a.pages + b.j) * TILE + (pos & 63)) * a.head_dim;
    paired_order = false;
    if (pos >= b.base + b.valid) return nullptr;
    return a.k_own + (((size_t)b.seq * a.kv_heads + b.h) * a.own_cap + (pos - a.prefix)) *
                         a.head_dim;
}
__device__ __forceinline__ const int16_t* q_row(const SharedAttnArgs& a, uint32_t h,
                                                uint32_t rho) {
    const uint32_t seq = rho / a.group, head = h * a.group + rho % a.group;
    return a.q + ((size_t)seq * a.kv_heads * a.group + head) * a.head_dim;
}

// The score by the definition: four banks of AP_RND-narrowed products, each
// saturating as its products arrive.
__device__ __noinline__ int32_t defined_score(const int16_t* q, const int16_t* k, bool paired_order,
                                              uint32_t d, int32_t qk_scale) {
    int32_t bank[4] = {0, 0, 0, 0};
    for (uint32_t e = 0; e < d; e += 4) {
#pragma unroll
        for (uint32_t u = 0; u < 4; u++) {
            const int32_t kv = k[paired_order ? paired(e + u) : e + u];
            const int32_t t = (int32_t)fx_rnd((int64_t)q[e + u] * fx_fm_to_wt(kv), 4);
            bank[u] = fx_sat32((int64_t)bank[u] + t);
        }
    }
    int32_t t = fx_sat32((int64_t)bank[0] + bank[1] + bank[2] + bank[3]);
    t = fx_sat32(fx_rnd((int64_t)t * ((int64_t)qk_scale << 8), 16));
    return fx_sat16(fx_rnd(t, 8));
}

// Scores of the job's rows.  KC: 64-element chunks of a head.
template <int KC, bool OWN>
__device__ __forceinline__ void score_job(const SharedAttnArgs& a, const Job& b) {
    const uint32_t lane = threadIdx.x & 63, q = lane & 15, g = lane >> 4, d = a.head_dim;
    const v4i zero = {0, 0, 0, 0};
    // all K rows of the tile: strip s holds positions 16 s .. + 15
    v4u raw[4][KC][2];
    bool natural[4];
#pragma unroll
    for (int s = 0; s < 4; s++) {
        bool pr;
        const int16_t* row = k_row(a, b, b.base + 16 * s + q, pr);
        natural[s] = !pr;
#pragma unroll
        for (int kc = 0; kc < KC; kc++) {
            const uint32_t e = 64 * kc + 16 * g;
            raw[s][kc][0] = raw[s][kc][1] = v4u{0, 0, 0, 0};
            if (e < d && (!OWN || row)) {
                raw[s][kc][0] = *(const v4u*)(row + e);
                raw[s][kc][1] = *(const v4u*)(row + e + 8);
            }
        }
    }
    v4i ka[4][KC], kb[4][KC], bias[4];
    uint32_t any = 0;
    const v4i ones = {0x01010101, 0x01010101, 0x01010101, 0x01010101};
#pragma unroll
    for (int s = 0; s < 4; s++) {
        v4i sa = zero, sb = zero;
#pragma unroll
        for (int kc = 0; kc < KC; kc++) {
            v4u x = raw[s][kc][0], y = raw[s][kc][1];
            if (OWN && natural[s]) x = pair8(x), y = pair8(y);
            planes16(x, y, ka[s][kc], kb[s][kc], any);
            sa = mfma16(ka[s][kc], ones, sa);
            sb = mfma16(kb[s][kc], ones, sb);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) bias[s][i] = 128 * (256 * sa[i] + sb[i]);
    }
    const bool kf = __any(any != 0);
    for (uint32_t r0 = b.rho; r0 < b.end; r0 += 16) {
        const uint32_t rho = min(r0 + q, b.end - 1);  // rows past the last repeat it
        const bool real = r0 + q < b.end;
        const int16_t* qr = q_row(a, b.h, rho);
        v4i qc[KC], qd[KC], qh[KC], ql[KC];
        uint32_t low = 0xf;  // banks whose queries are all -32768
#pragma unroll
        for (int kc = 0; kc < KC; kc++) {
            const uint32_t e = 64 * kc + 16 * g;
            v4u x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
            if (e < d) {
                x = pair8(*(const v4u*)(qr + e));
                y = pair8(*(const v4u*)(qr + e + 8));
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (x[i] != 0x80008000u || y[i] != 0x80008000u) low &= ~(1u << i);
            qc[kc] = v4i{(int32_t)plane_c(x.x, x.y), (int32_t)plane_c(x.z, x.w),
                         (int32_t)plane_c(y.x, y.y), (int32_t)plane_c(y.z, y.w)};
            qd[kc] = v4i{(int32_t)plane_d(x.x, x.y), (int32_t)plane_d(x.z, x.w),
                         (int32_t)plane_d(y.x, y.y), (int32_t)plane_d(y.z, y.w)};
            if (kf) corr_planes16(x, y, qh[kc], ql[kc]);
        }
        int32_t sc[4][4];
        // only 32 products of -32768 and -2048 pass a bank's 2^31 - 1
        low &= __shfl_xor(low, 16, 64);
        low &= __shfl_xor(low, 32, 64);
        if (d == 128 && __any(low != 0)) {
#pragma unroll 1
            for (int s = 0; s < 4; s++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    bool pr;
                    const int16_t* row = k_row(a, b, b.base + 16 * s + 4 * g + i, pr);
                    const int32_t v = OWN && !row ? 0 : defined_score(qr, row, pr, d, a.qk_scale);
#pragma unroll
                    for (int u = 0; u < 4; u++)
                        if (u == s) sc[u][i] = v;
                }
        } else {
#pragma unroll
            for (int s = 0; s < 4; s++) {
                v4i ac = zero, x = zero, bd = zero, mh = zero, ml = zero;
#pragma unroll
                for (int kc = 0; kc < KC; kc++) {
                    ac = mfma16(ka[s][kc], qc[kc], ac);
                    x = mfma16(ka[s][kc], qd[kc], x);
                    bd = mfma16(kb[s][kc], qd[kc], bd);
                    x = mfma16(kb[s][kc], qc[kc], x);
                    if (kf) {
                        const v4i mk = mask2048(ka[s][kc], kb[s][kc]);
                        mh = mfma16(mk, qh[kc], mh);
                        ml = mfma16(mk, ql[kc], ml);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    // sum = 256 t + lo; the two roundings of sum * scale are
                    // floor((sum qk + 2^7 + 2^15) / 2^16) in one, and a t past
                    // 2^23 (a sum past 32 bits) saturates the score
                    const int32_t l = bd[i] + bias[s][i] + ml[i];
                    const int32_t t = (ac[i] << 8) + x[i] + mh[i] + (l >> 8);
                    const int32_t lo = __mul24(l & 255, a.qk_scale) + 32896;
                    const int32_t v = __mul24(med3(t, -(1 << 23), (1 << 23) - 1), a.qk_scale) +
                                      (lo >> 8);
                    sc[s][i] = med3(v >> 8, INT16_MIN, INT16_MAX);
                }
            }
        }
        int32_t mx = INT16_MIN;
        int16_t* out = a.scores + (((size_t)b.h * a.tiles + b.j) * a.rows_pad + rho) * TILE;
#pragma unroll
        for (int s = 0; s < 4; s++) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (OWN && 16 * s + 4 * g + i >= b.valid) sc[s][i] = INT16_MIN;
                mx = max(mx, sc[s][i]);
            }
            if (real)
                *(v2u*)(out + 16 * s + 4 * g) =
                    v2u{pack16(sc[s][0], sc[s][1]), pack16(sc[s][2], sc[s][3])};
        }
        mx = quad_max(mx);
        if (real && g == 0)
            a.tmax[((size_t)b.h * a.rows_pad + rho) * a.tmax_ld + b.j] = (int16_t)mx;
    }
}

template <int KC>
__global__ __launch_bounds__(256, 2) void shared_scores_kernel(SharedAttnArgs a,
                                                               uint32_t shared_blocks) {
    Job b;
    if (!job_of(a, shared_blocks, b)) return;
    if (b.own)
        score_job<KC, true>(a, b);
    else
        score_job<KC, false>(a, b);
}

// LDS row of a head element of an own tile (positions bank-paired; 16 bytes
// past 64 positions, so that rows start in different banks).
constexpr uint32_t kOwnRow = 72;

// Elements [e0, e0 + ec) of the own tile's V rows into `vt` [ec][kOwnRow] by
// the calling wavefront (ec a multiple of 16).
__device__ __forceinline__ void own_values(const SharedAttnArgs& a, const Job& b, uint32_t e0,
                                           uint32_t ec, int16_t* vt) {
    const uint32_t lane = threadIdx.x & 63, d = a.head_dim;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // what was read from vt before
    __builtin_amdgcn_wave_barrier();
    // positions of the tile that lie in the prefix: its last page's
    const uint32_t head = b.base < a.prefix ? a.prefix - b.base : 0;  // < 64
    if (head) {
        const int16_t* page = a.vcache + (((size_t)b.h * a.pages + b.j) * d + e0) * TILE;
        for (uint32_t i = lane; i < 8 * ec; i += 64)  // 8 positions of an element
            *(v4u*)(vt + (i >> 3) * kOwnRow + 8 * (i & 7)) = *(const v4u*)(page + 8 * i);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    const int16_t* own = a.v_own + ((size_t)b.seq * a.kv_heads + b.h) * a.own_cap * d + e0;
    // positions p and p + 4 of a group of 8, 8 elements at a time
    const uint32_t per = ec / 8;
    for (uint32_t i = lane; i < 32 * per; i += 64) {
        const uint32_t pr = i / per, e = 8 * (i % per);
        const uint32_t p0 = 8 * (pr >> 2) + (pr & 3), p1 = p0 + 4;
        if (p1 < head) continue;
        v4u x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
        if (p0 >= head && p0 < b.valid)
            x = *(const v4u*)(own + (size_t)(b.base + p0 - a.prefix) * d + e);
        if (p1 < b.valid) y = *(const v4u*)(own + (size_t)(b.base + p1 - a.prefix) * d + e);
        int16_t* o = vt + e * kOwnRow + 8 * (pr >> 2) + 2 * (pr & 3);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const uint32_t w0 = __builtin_amdgcn_perm(y[u], x[u], 0x05040100u);
            const uint32_t w1 = __builtin_amdgcn_perm(y[u], x[u], 0x07060302u);
            if (p0 >= head) {
                *(uint32_t*)(o + (2 * u) * kOwnRow) = w0;
                *(uint32_t*)(o + (2 * u + 1) * kOwnRow) = w1;
            } else {  // p0 is the prefix's
                o[(2 * u) * kOwnRow + 1] = (int16_t)(w0 >> 16);
                o[(2 * u + 1) * kOwnRow + 1] = (int16_t)(w1 >> 16);
            }
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Values of the job's rows.  NE: 16-element strips of a head, rounded up.
template <int NE, bool OWN>
__device__ __forceinline__ void value_job(const SharedAttnArgs& a, const Job& b,
                                          const int16_t* e14, int16_t* vt) {
    const uint32_t lane = threadIdx.x & 63, q = lane & 15, g = lane >> 4, d = a.head_dim;
    const uint32_t ne = d / 16;
    v4i va[NE], vb[NE];
    uint32_t any = 0;
    {
        v4u raw[NE][2];
        const int16_t* page = a.vcache + ((size_t)b.h * a.pages + b.j) * TILE * d;
#pragma unroll
        for (int es = 0; es < NE; es++) {
            // strips past the head's repeat its last
            const uint32_t strip = min((uint32_t)es, ne - 1);
            if (OWN && es % 4 == 0 && es < (int)ne)
                own_values(a, b, 16 * es, min(64u, d - 16 * es), vt);
            const uint32_t e = 16 * strip + q;
            const int16_t* p = OWN ? vt + (e & 63) * kOwnRow + 16 * g : page + e * TILE + 16 * g;
            raw[es][0] = *(const v4u*)p;
            raw[es][1] = *(const v4u*)(p + 8);
        }
#pragma unroll
        for (int es = 0; es < NE; es++) planes16(raw[es][0], raw[es][1], va[es], vb[es], any);
    }
    const bool vf = __any(any != 0);
    const v4i zero = {0, 0, 0, 0};
    for (uint32_t r0 = b.rho; r0 < b.end; r0 += 16) {
        const uint32_t rho = min(r0 + q, b.end - 1);
        const bool real = r0 + q < b.end;
        const size_t row = ((size_t)b.h * a.tiles + b.j) * a.rows_pad + rho;
        const v4u s0 = *(const v4u*)(a.scores + row * TILE + 16 * g);
        const v4u s1 = *(const v4u*)(a.scores + row * TILE + 16 * g + 8);
        // the running maximum before this tile, and with it
        const int16_t* tm = a.tmax + ((size_t)b.h * a.rows_pad + rho) * a.tmax_ld;
        int32_t before = INT16_MIN;
        for (uint32_t t = 8 * g; t < b.j; t += 32) {
            const v4u w = *(const v4u*)(tm + t);
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const int32_t m = half16(w, u);
                if (t + u < b.j) before = max(before, m);
            }
        }
        before = quad_max(before);
        const int32_t top = max(before, (int32_t)tm[b.j]);
        int32_t p[16], sum = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int32_t s = i < 8 ? half16(s0, i) : half16(s1, i - 8);
            const int32_t e = e14[max(s - top, -2048) + 2048];
            p[i] = !OWN || 16 * g + i < b.valid ? e : 0;
            sum += p[i];
        }
        sum = quad_sum(sum);
        if (real && g == 0) {
            a.old[row] = (int32_t)e14[max(before - top, -2048) + 2048] << 2;
            a.tsum[row] = sum << 2;
        }
        // bank-paired words (p, p + 4) of each group of 8
        v4i pc, pd, ph, pl;
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int at = 8 * (i >> 2) + (i & 3);
            w[i] = pack16(p[at], p[at + 4]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            // p + 128 <= 16512: no carry between the halves
            pc[i] = (int32_t)plane_c(w[2 * i] + 0x00800080u, w[2 * i + 1] + 0x00800080u);
            pd[i] = (int32_t)low_plane(w[2 * i], w[2 * i + 1]);
        }
        ph = pl = zero;
        if (vf)
            corr_planes16(v4u{w[0], w[1], w[2], w[3]}, v4u{w[4], w[5], w[6], w[7]}, ph, pl);
        int16_t* out = a.tval + row * d + 4 * g;
#pragma unroll
        for (int es = 0; es < NE; es++) {
            v4i ac = mfma16(va[es], pc, zero);
            v4i x = mfma16(va[es], pd, zero);
            v4i bd = mfma16(vb[es], pd, zero);
            x = mfma16(vb[es], pc, x);
            if (vf) {
                const v4i mk = mask2048(va[es], vb[es]);
                x = mfma16(mk, ph, x);
                bd = mfma16(mk, pl, bd);
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
                tv[i] = med3((int32_t)(tot + 8224) >> 14, INT16_MIN, INT16_MAX);
            }
            if (real && es < (int)ne)
                *(v2u*)(out + 16 * es) = v2u{pack16(tv[0], tv[1]), pack16(tv[2], tv[3])};
        }
    }
}

template <int NE>
__global__ __launch_bounds__(256, 2) void shared_values_kernel(SharedAttnArgs a,
                                                               uint32_t shared_blocks) {
    __shared__ __attribute__((aligned(16))) int16_t e14[2056];
    __shared__ __attribute__((aligned(16))) int16_t vt[4][64 * kOwnRow];
    for (uint32_t i = threadIdx.x; i < 257; i += 256)
        *(v4u*)(e14 + 8 * i) = *(const v4u*)(a.exp14 + 8 * i);
    __syncthreads();
    Job b;
    if (!job_of(a, shared_blocks, b)) return;
    if (b.own)
        value_job<NE, true>(a, b, e14, vt[threadIdx.x >> 6]);
    else
        value_job<NE, false>(a, b, e14, nullptr);
}

// Two elements of a row per thread: the chain over its tiles, eight tiles'
// operands requested together.
__global__ __launch_bounds__(256) void shared_join_kernel(SharedAttnArgs a) {
    const uint32_t half = a.head_dim / 2, id = blockIdx.x * 256 + threadIdx.x;
    const uint32_t e = 2 * (id % half), row = id / half;
    if (row >= a.kv_heads * a.rows) return;
    const uint32_t h = row / a.rows, rho = row % a.rows;
    const uint32_t n = a.prefix + length_of(a, rho / a.group), nt = (n + 63) / 64;
    int32_t sum = 0, acc0 = 0, acc1 = 0;
    const size_t step = a.rows_pad, at = (size_t)h * a.tiles * step + rho;
    const int32_t* po = a.old + at;
    const int32_t* ps = a.tsum + at;
    const int16_t* pv = a.tval + at * a.head_dim + e;
    constexpr uint32_t U = 8;
    for (uint32_t t0 = 0; t0 < nt; t0 += U) {
        int32_t old[U], ts[U];
        uint32_t v[U];
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const size_t t = min(t0 + u, nt - 1);
            old[u] = po[t * step];
            ts[u] = ps[t * step];
            v[u] = *(const uint32_t*)(pv + t * step * a.head_dim);
        }
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            if (t0 + u >= nt) break;
            if (__any(old[u] != 65536)) {  // else the factors are 1.0
                sum = rnd16_mul(sum, old[u]);
                acc0 = rnd16_mul(acc0, old[u]);
                acc1 = rnd16_mul(acc1, old[u]);
            }
            sum = __builtin_elementwise_add_sat(sum, ts[u]);
            acc0 = __builtin_elementwise_add_sat(acc0, (int32_t)(int16_t)(v[u] & 0xffffu) << 8);
            acc1 = __builtin_elementwise_add_sat(acc1, ((int32_t)v[u] >> 16) << 8);
        }
    }
    const int32_t inv = fx_inv_sum(sum);
    const size_t head = (size_t)(rho / a.group) * a.kv_heads * a.group + h * a.group +
                        rho % a.group;
    *(uint32_t*)(a.out + head * a.head_dim + e) =
        pack16(sat16_32(rnd16_mul(acc0, inv)), sat16_32(rnd16_mul(acc1, inv)));
}

uint32_t round_to(uint32_t v, uint32_t m) { return (v + m - 1) / m * m; }
size_t part_bytes(size_t n) { return (n + 255) / 256 * 256; }

template <int NE>
hipError_t launch_values(const SharedAttnArgs& a, uint32_t grid, uint32_t shared_blocks,
                         hipStream_t st) {
    shared_values_kernel<NE><<<grid, 256, 0, st>>>(a, shared_blocks);
    return hipGetLastError();
}

}  // namespace

void shared_attention_shape(SharedAttnArgs& a) {
    a.whole = a.prefix / 64;
    const uint32_t tail = a.prefix % 64 + a.own_cap;
    a.own_tiles = (tail + 63) / 64;
    a.tiles = a.whole + a.own_tiles;
    a.tmax_ld = round_to(a.tiles, 32);
    a.rows = a.sequences * a.group;
    a.rows_pad = round_to(a.rows, 16);
    // A wavefront converts a tile's K (V) once for the pieces it takes: as
    // many as leave a tile four wavefronts, at most four.
    const uint32_t pieces = a.rows_pad / 16;
    a.per_wave = pieces / 4 < 1 ? 1 : (pieces / 4 > 4 ? 4 : pieces / 4);
    a.groups = (pieces + a.per_wave - 1) / a.per_wave;
    a.shared_jobs = a.kv_heads * a.whole * a.groups;
    a.own_jobs = a.kv_heads * a.sequences * a.own_tiles;
}

size_t shared_attention_bytes(const SharedAttnArgs& a) {
    const size_t rt = (size_t)a.kv_heads * a.tiles * a.rows_pad;
    return part_bytes(rt * 64 * 2) + part_bytes((size_t)a.kv_heads * a.rows_pad * a.tmax_ld * 2) +
           2 * part_bytes(rt * 4) + part_bytes(rt * a.head_dim * 2);
}

void shared_attention_scratch(SharedAttnArgs& a, uint8_t* base) {
    const size_t rt = (size_t)a.kv_heads * a.tiles * a.rows_pad;
    auto take = [&](size_t bytes) {
        uint8_t* p = base;
        base += part_bytes(bytes);
        return p;
    };
    a.scores = (int16_t*)take(rt * 64 * 2);
    a.tmax = (int16_t*)take((size_t)a.kv_heads * a.rows_pad * a.tmax_ld * 2);
    a.old = (int32_t*)take(rt * 4);
    a.tsum = (int32_t*)take(rt * 4);
    a.tval = (int16_t*)take(rt * a.head_dim * 2);
}

hipError_t launch_shared_attention(const SharedAttnArgs& a, hipStream_t st) {
    const uint32_t shared_blocks = (a.shared_jobs + 3) / 4;
    const uint32_t grid = shared_blocks + (a.own_jobs + 3) / 4;
    if (grid) {
        if (a.head_dim <= 64)
            shared_scores_kernel<1><<<grid, 256, 0, st>>>(a, shared_blocks);
        else
            shared_scores_kernel<2><<<grid, 256, 0, st>>>(a, shared_blocks);
        hipError_t e = hipGetLastError();
        if (e == hipSuccess)
            e = a.head_dim <= 64 ? launch_values<4>(a, grid, shared_blocks, st)
                                 : launch_values<8>(a, grid, shared_blocks, st);
        if (e != hipSuccess) return e;
    }
    const uint32_t threads = a.kv_heads * a.rows * (a.head_dim / 2);
    shared_join_kernel<<<(threads + 255) / 256, 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace llm
