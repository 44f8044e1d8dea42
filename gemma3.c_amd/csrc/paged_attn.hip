// paged_attn.hip - attention of many sequences over a KV cache in pages, on
// MFMA (gfx950): packed prompts (paged_prefill) and one query per sequence
// with shared prefixes (paged_decode).
//
// o_i = sum_j p_ij v_j / sum_j p_ij, p_ij = exp(q_i . k_j / 16), over the
// positions j that query i sees: (pos_i - window, pos_i].
//
// Precision.  q, the outputs and fp32 pages hold 24 bits, no MFMA input
// format does.  Every operand x is scaled by a power of two and split,
// x = hi + lo, hi = fp16(x), lo = fp16(x - hi): 22 bits, and with the largest
// magnitude of its block scaled to [2^13, 2^14) an absolute floor 2^-38 of it
// for the small ones.  A product is hi.hi + hi.lo + lo.hi in fp32; the
// dropped lo.lo is 2^-22 of it.  bf16 pages are exact in the hi plane alone,
// which leaves two products.  So the matrix units do 3x (2x) the algorithmic
// work.  Scores, maxima, sums and accumulators are fp32.
//
// One workgroup = 4 waves = one KV head x 64 MT query rows (a row is one
// query head of one token; the heads of a group share the keys); each wave
// owns 16 MT rows over the full head dim (MT blocks: Q hi / lo 64 VGPRs, O^T
// 64 each) and walks 32-key tiles that the four waves load and convert
// together:
//   S^T[key][row] = K . Q^T,  O^T[dim][row] += V^T . P^T,
// both v_mfma_f32_16x16x32_f16.  In the 16x16 accumulator lane l holds column
// (row) l % 16, so a row's softmax state lives in the lanes l % 16 + 16 g.
//
// LDS holds a tile as MFMA A operands in lane order (1 KiB each, so every
// read is one conflict-free ds_read_b128): K [2 key blocks][8 dim steps], V
// [16 dim blocks], each hi then lo.  Wave w brings keys 4w..4w+3 and
// 16+4w..16+4w+3, one coalesced row per load.  These are the keys lane group
// g = w of the S^T registers holds, so P goes from the S^T registers to the
// P.V operand without a shuffle, and one scale per wave and tile is one
// factor per lane group: K's on the scores, V's on P.  A V lane holds 4 dims
// of the 8 keys, which are whole operand lanes of the four dim blocks
// {64 T + 4 c + t}: the transposition is register naming.  K lanes write half
// an operand lane (4 dims) each, at a position XORed by the dim step, so the
// 8-byte stores spread over the banks.
#include <hip/hip_runtime.h>
#include <limits.h>

#include "g3k.h"
#include "g3k_device.h"
#include "paged_body.h"

namespace {

using namespace g3k;

constexpr int D = G3K_HEAD_DIM;
constexpr int BK = 32;                      // keys per tile
constexpr float M_NONE = -3.402823466e38f;  // running max before any key
constexpr int E_NONE = -1000;               // running V exponent before any tile
constexpr float LAZY = 8.0f;                // log2 headroom of the lazy max
constexpr int P_EXP = 6;                    // P is scaled by 2^P_EXP: p <= 2^LAZY stays below 2^14
constexpr int X_EXP = 14;                   // q, K, V: largest magnitude of a block below 2^X_EXP

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half4v __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mfma(half8 a, half8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ half2v cvt2(float a, float b) { return __builtin_convertvector((f32x2){a, b}, half2v); }

// The power-of-two exponent of a block whose largest magnitude is m: m <
// 2^exponent.  A block of zeros, or of values below 2^-100, counts as 2^-100;
// one with an infinity or NaN as 2^127 (its rows come out as they may).
__device__ __forceinline__ int block_exponent(float m) {
    if (!(m < INFINITY)) return 127;
    const int e = __builtin_amdgcn_frexp_expf(m);
    return m == 0.f || e < -100 ? -100 : e;
}

// x s as hi + lo, two values at a time.
__device__ __forceinline__ void split2(float a, float b, float s, half2v &hi, half2v &lo) {
    hi = cvt2(a * s, b * s);
    lo = cvt2(__builtin_fmaf(a, s, -(float)hi.x), __builtin_fmaf(b, s, -(float)hi.y));
}

// What a workgroup attends: query rows row0.. of a run of tokens over keys
// [kbeg, kend) of table row b.
struct Unit {
    int b, kbeg, kend;
    int first, count;      // rows (of the group's heads): the first row's index among the run's, and how many
    int run;               // prefill: packed row of the run's first token; decode: the run's first sequence
    int pos;               // prefill: position of that token
};

// ---- the tile walk -----------------------------------------------------------

template <bool BF16>
struct Lds {
    static constexpr int PL = BF16 ? 1 : 2;            // planes
    static constexpr int K_BYTES = 2 * 8 * PL * 1024;  // [key block][dim step][plane] operands
    static constexpr int V_BYTES = 16 * PL * 1024;     // [dim block][plane]
    static constexpr int BUF = K_BYTES + V_BYTES;
    static constexpr int BYTES = 2 * BUF;
};

// One tile's rows in flight: this wave's 8 keys, 4 dims a lane.
template <bool BF16>
struct Raw;
template <>
struct Raw<false> {
    f32x4 k[8], v[8];
};
template <>
struct Raw<true> {
    u32x2 k[8], v[8];
};

template <bool BF16>
__device__ __forceinline__ void unpack(const Raw<BF16> &r, int i, bool v, float x[4]) {
    if constexpr (BF16) {
        const u32x2 u = v ? r.v[i] : r.k[i];
        x[0] = __uint_as_float(u.x << 16);
        x[1] = __uint_as_float(u.x & 0xffff0000u);
        x[2] = __uint_as_float(u.y << 16);
        x[3] = __uint_as_float(u.y & 0xffff0000u);
    } else {
        const f32x4 u = v ? r.v[i] : r.k[i];
        x[0] = u.x;
        x[1] = u.y;
        x[2] = u.z;
        x[3] = u.w;
    }
}

// Where a tile's rows are: element offsets of this wave's 8 rows from the
// head's first page row, and which of its two runs of 4 keys have no page.
struct Place {
    long long off[8];
    int bad;
};

// Keys outside [kbeg, kend) take the nearest row inside, so nothing else is
// read; their scores are masked.  A table entry outside the pool is never
// followed: its run reads page 0 and is then zeroed and masked.
__device__ __forceinline__ Place place_tile(const g3k_paged_args &a, const int *table, int tile, int wave, int kbeg,
                                            int kend) {
    Place p;
    p.bad = 0;
    const int j0 = tile * BK;
    const int mask = (1 << a.s.page_shift) - 1;
    if (j0 >= kbeg && j0 + BK <= kend) {
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int j = j0 + 16 * c + 4 * wave;
            int page = __builtin_amdgcn_readfirstlane(table[j >> a.s.page_shift]);
            if ((unsigned)page >= (unsigned)a.num_pages) {
                page = 0;
                p.bad |= 1 << c;
            }
            const long long o = page * a.page_stride + (long long)(j & mask) * D;
#pragma unroll
            for (int i = 0; i < 4; i++) p.off[4 * c + i] = o + i * D;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int j = clampi(j0 + 16 * (i >> 2) + 4 * wave + (i & 3), kbeg, kend - 1);
            int page = __builtin_amdgcn_readfirstlane(table[j >> a.s.page_shift]);
            if ((unsigned)page >= (unsigned)a.num_pages) {
                page = 0;
                p.bad |= 1 << (i >> 2);
            }
            p.off[i] = page * a.page_stride + (long long)(j & mask) * D;
        }
    }
    return p;
}

template <bool BF16>
__device__ __forceinline__ void load_tile(const void *k, const void *v, const Place &p, int lane, Raw<BF16> &r) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if constexpr (BF16) {
            r.k[i] = *reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(k) + p.off[i] + 4 * lane);
        } else {
            r.k[i] = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(k) + p.off[i] + 4 * lane);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if constexpr (BF16) {
            r.v[i] = *reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(v) + p.off[i] + 4 * lane);
        } else {
            r.v[i] = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(v) + p.off[i] + 4 * lane);
        }
    }
}

// Splits the rows in flight into operands and stores them, with the wave's
// factors: {K's factor on the scores, the two runs' additive masks, V's
// exponent}.
template <bool BF16>
__device__ __forceinline__ void store_tile(Raw<BF16> &r, int bad, char *buf, f32x4 *factors, int wave, int lane) {
    using L = Lds<BF16>;
    if (bad) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if ((bad >> (i >> 2)) & 1) {
                r.k[i] = 0;
                r.v[i] = 0;
            }
    }
    float mk = 0.f, mv = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float x[4];
        unpack<BF16>(r, i, false, x);
        mk = fmaxf(mk, fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
        unpack<BF16>(r, i, true, x);
        mv = fmaxf(mv, fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
    }
    const int ek = block_exponent(wave_max(mk)), ev = block_exponent(wave_max(mv));
    const float sk = __builtin_amdgcn_ldexpf(1.0f, X_EXP - ek), sv = __builtin_amdgcn_ldexpf(1.0f, X_EXP - ev);
    if (lane == 0)
        factors[wave] = (f32x4){__builtin_amdgcn_ldexpf(1.0f, ek - X_EXP), bad & 1 ? -INFINITY : 0.f,
                                bad & 2 ? -INFINITY : 0.f, __int_as_float(ev)};
    // K: lane holds dims 4 lane.. = half (lane & 1) of operand lane group
    // (lane >> 1) & 3 of dim step lane >> 3
    char *kd = buf + (lane >> 3) * (L::PL * 1024) + ((lane >> 1) & 3) * 256 + (lane & 1) * 8;
    const int f = (lane >> 1) & 15;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float x[4];
        unpack<BF16>(r, i, false, x);
        char *d = kd + (i >> 2) * (8 * L::PL * 1024) + (((4 * wave + (i & 3)) ^ f) << 4);
        half4v h, l;
        if constexpr (BF16) {
            h.xy = cvt2(x[0] * sk, x[1] * sk);
            h.zw = cvt2(x[2] * sk, x[3] * sk);
        } else {
            half2v a, b;
            split2(x[0], x[1], sk, a, b);
            h.xy = a;
            l.xy = b;
            split2(x[2], x[3], sk, a, b);
            h.zw = a;
            l.zw = b;
            *reinterpret_cast<half4v *>(d + 1024) = l;
        }
        *reinterpret_cast<half4v *>(d) = h;
    }
    // V: lane holds dims 4 lane + t of the 8 keys = operand lane lane & 15 of
    // group `wave` of dim blocks 4 (lane >> 4) + t
    char *vd = buf + L::K_BYTES + (lane >> 4) * (4 * L::PL * 1024) + wave * 256 + (lane & 15) * 16;
    float x[8][4];
#pragma unroll
    for (int i = 0; i < 8; i++) unpack<BF16>(r, i, true, x[i]);
#pragma unroll
    for (int t = 0; t < 4; t++) {
        half8 h, l;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            half2v hh, ll;
            if constexpr (BF16) {
                hh = cvt2(x[i][t] * sv, x[i + 1][t] * sv);
            } else {
                split2(x[i][t], x[i + 1][t], sv, hh, ll);
                l[i] = ll.x;
                l[i + 1] = ll.y;
            }
            h[i] = hh.x;
            h[i + 1] = hh.y;
        }
        *reinterpret_cast<half8 *>(vd + t * (L::PL * 1024)) = h;
        if constexpr (!BF16) *reinterpret_cast<half8 *>(vd + t * (L::PL * 1024) + 1024) = l;
    }
}

// The rows of a wave: queries in registers, running softmax state, O^T.
template <int MT>
struct Rows {
    half8 qh[MT][8], ql[MT][8];
    f32x4 o[MT][16];
    float factor[MT], m[MT], l[MT];   // l: this lane's keys only
    int lo[MT], hi[MT];               // the keys this lane's row sees
    int lo_min, lo_max, hi_min, hi_max;   // over the wave's rows
    int ev;                           // O^T's exponent: o = true o * 2^(X_EXP + P_EXP - ev), unnormalised
};

template <int MT>
__device__ __forceinline__ void load_query(const float *q, bool live, float qscale, int mt, int lane, Rows<MT> &s) {
    float x[8][8];
    float m = 0.f;
#pragma unroll
    for (int kk = 0; kk < 8; kk++) {
        const f32x4 z = {0.f, 0.f, 0.f, 0.f};
        const float *p = q + 32 * kk + 8 * (lane >> 4);
        const f32x4 a = live ? *reinterpret_cast<const f32x4 *>(p) : z;
        const f32x4 b = live ? *reinterpret_cast<const f32x4 *>(p + 4) : z;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[kk][i] = a[i];
            x[kk][4 + i] = b[i];
            m = fmaxf(m, fmaxf(fabsf(a[i]), fabsf(b[i])));
        }
    }
    const int e = block_exponent(col4_max(m));
    const float sc = __builtin_amdgcn_ldexpf(1.0f, X_EXP - e);
    s.factor[mt] = __builtin_amdgcn_ldexpf(qscale, e - X_EXP);
#pragma unroll
    for (int kk = 0; kk < 8; kk++)
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            half2v h, l;
            split2(x[kk][i], x[kk][i + 1], sc, h, l);
            s.qh[mt][kk][i] = h.x;
            s.qh[mt][kk][i + 1] = h.y;
            s.ql[mt][kk][i] = l.x;
            s.ql[mt][kk][i + 1] = l.y;
        }
}

// One tile's keys for the wave's rows.
template <bool BF16, int MT>
__device__ __forceinline__ void attend_tile(const char *buf, const f32x4 *factors, int tile, int lane, Rows<MT> &s) {
    using L = Lds<BF16>;
    const int j0 = tile * BK;
    const int g = lane >> 4, c = lane & 15;
    f32x4 sc[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) sc[mt][0] = sc[mt][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < 8; kk++) {
        const char *kp = buf + kk * (L::PL * 1024) + g * 256 + ((c ^ ((4 * kk + g) & 15)) << 4);
        half8 kh[2], kl[2];
#pragma unroll
        for (int kt = 0; kt < 2; kt++) {
            kh[kt] = *reinterpret_cast<const half8 *>(kp + kt * (8 * L::PL * 1024));
            if constexpr (!BF16) kl[kt] = *reinterpret_cast<const half8 *>(kp + kt * (8 * L::PL * 1024) + 1024);
        }
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int mt = 0; mt < MT; mt++) sc[mt][kt] = mfma(kh[kt], s.qh[mt][kk], sc[mt][kt]);
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int mt = 0; mt < MT; mt++) sc[mt][kt] = mfma(kh[kt], s.ql[mt][kk], sc[mt][kt]);
        if constexpr (!BF16) {
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int mt = 0; mt < MT; mt++) sc[mt][kt] = mfma(kl[kt], s.qh[mt][kk], sc[mt][kt]);
        }
    }
    const f32x4 fac = factors[g];
    const int ev = __float_as_int(fac.w);
    // the tile's V exponent, over the four lane groups
    const int ev_tile = max(max(__float_as_int(factors[0].w), __float_as_int(factors[1].w)),
                            max(__float_as_int(factors[2].w), __float_as_int(factors[3].w)));
    const bool ragged = j0 < s.lo_max || j0 + BK > s.hi_min;
    float tmax[MT];
    bool grow = ev_tile > s.ev;
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const float f = s.factor[mt] * fac.x;
        float t = M_NONE;
#pragma unroll
        for (int kt = 0; kt < 2; kt++) {
            const float bias = kt ? fac.z : fac.y;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float x = __builtin_fmaf(sc[mt][kt][r], f, bias);
                if (ragged) {
                    const int j = j0 + 16 * kt + 4 * g + r;
                    if (j < s.lo[mt] || j >= s.hi[mt]) x = -INFINITY;
                }
                sc[mt][kt][r] = x;
                t = fmaxf(t, x);
            }
        }
        tmax[mt] = col4_max(t);
        grow |= tmax[mt] > s.m[mt] + LAZY;
    }
    // O^T and l are rescaled when a row's max outgrows its reference by
    // 2^LAZY, or V's exponent the one O^T is held at (two bits above what it
    // was first, so ordinary tiles do not move it)
    if (__builtin_amdgcn_ballot_w64(grow)) {
        const int e = ev_tile > s.ev ? ev_tile + 2 : s.ev;
        const float down = s.ev == E_NONE ? 0.f : __builtin_amdgcn_ldexpf(1.0f, s.ev - e);
        s.ev = e;
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const float m = tmax[mt] > s.m[mt] + LAZY ? tmax[mt] : s.m[mt];
            const float keep = fast_exp2(s.m[mt] - m);
            s.m[mt] = m;
            s.l[mt] *= keep;
            const float x = keep * down;
#pragma unroll
            for (int d = 0; d < 16; d++) s.o[mt][d] *= x;
        }
    }
    const float pf = __builtin_amdgcn_ldexpf(1.0f, P_EXP + ev - s.ev);
    half8 ph[MT], pl[MT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                const float a = fast_exp2(sc[mt][kt][r] - s.m[mt]), b = fast_exp2(sc[mt][kt][r + 1] - s.m[mt]);
                s.l[mt] += a + b;
                half2v h, l;
                split2(a, b, pf, h, l);
                ph[mt][4 * kt + r] = h.x;
                ph[mt][4 * kt + r + 1] = h.y;
                pl[mt][4 * kt + r] = l.x;
                pl[mt][4 * kt + r + 1] = l.y;
            }
    }
    const char *vp = buf + L::K_BYTES + lane * 16;
#pragma unroll
    for (int d = 0; d < 16; d++) {
        const half8 vh = *reinterpret_cast<const half8 *>(vp + d * (L::PL * 1024));
#pragma unroll
        for (int mt = 0; mt < MT; mt++) s.o[mt][d] = mfma(vh, ph[mt], s.o[mt][d]);
#pragma unroll
        for (int mt = 0; mt < MT; mt++) s.o[mt][d] = mfma(vh, pl[mt], s.o[mt][d]);
        if constexpr (!BF16) {
            const half8 vl = *reinterpret_cast<const half8 *>(vp + d * (L::PL * 1024) + 1024);
#pragma unroll
            for (int mt = 0; mt < MT; mt++) s.o[mt][d] = mfma(vl, ph[mt], s.o[mt][d]);
        }
    }
}

// The whole walk of a workgroup over its unit's tiles.  Tile t + 1 is split
// and stored while tile t + 2 is fetched, then tile t is attended: one
// barrier a tile, and a fetch has a whole tile's work to arrive.
template <bool BF16, int MT>
__device__ __forceinline__ void walk(const g3k_paged_args &a, int head, const Unit &u, char *lds, f32x4 *factors, int wave,
                                     int lane, Rows<MT> &s) {
    using L = Lds<BF16>;
    const int t0 = u.kbeg / BK, t1 = u.kend > u.kbeg ? (u.kend + BK - 1) / BK : t0;
    if (t0 >= t1) return;
    const int *table = a.s.page_table + (long long)u.b * a.s.table_stride;
    const long long head_off = ((long long)head << a.s.page_shift) * D;
    const size_t es = BF16 ? 2 : 4;
    const void *kb = static_cast<const char *>(a.k) + head_off * es, *vb = static_cast<const char *>(a.v) + head_off * es;
    Raw<BF16> raw;
    Place p = place_tile(a, table, t0, wave, u.kbeg, u.kend);
    load_tile<BF16>(kb, vb, p, lane, raw);
    int bad = p.bad;
    store_tile<BF16>(raw, bad, lds, factors, wave, lane);
    if (t0 + 1 < t1) {
        p = place_tile(a, table, t0 + 1, wave, u.kbeg, u.kend);
        load_tile<BF16>(kb, vb, p, lane, raw);
        bad = p.bad;
    }
    // only LDS has to have arrived at these barriers: 63 vector memory
    // operations may stay in flight
    G3K_WAIT_BARRIER(63);
    for (int t = t0; t < t1; t++) {
        const int x = (t - t0) & 1;
        if (t + 1 < t1) {
            store_tile<BF16>(raw, bad, lds + (x ^ 1) * L::BUF, factors + 4 * (x ^ 1), wave, lane);
            if (t + 2 < t1) {
                p = place_tile(a, table, t + 2, wave, u.kbeg, u.kend);
                load_tile<BF16>(kb, vb, p, lane, raw);
                bad = p.bad;
            }
        }
        if (t * BK < s.hi_max && t * BK + BK > s.lo_min)
            attend_tile<BF16, MT>(lds + x * L::BUF, factors + 4 * x, t, lane, s);
        G3K_WAIT_BARRIER(63);
    }
}

// Row state before the walk, from the keys each lane's row sees: [lo, hi),
// or [0, INT_MAX) for a lane without a row.
template <int MT>
__device__ __forceinline__ void begin_rows(Rows<MT> &s) {
    int lo_min = INT_MAX, hi_max = 0, lo_max = 0, hi_min = INT_MAX;
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        s.m[mt] = M_NONE;
        s.l[mt] = 0.f;
#pragma unroll
        for (int d = 0; d < 16; d++) s.o[mt][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
        if (s.hi[mt] == INT_MAX) continue;      // not a row
        if (s.hi[mt] > s.lo[mt]) {
            lo_min = min(lo_min, s.lo[mt]);
            hi_max = max(hi_max, s.hi[mt]);
        }
        lo_max = max(lo_max, s.lo[mt]);
        hi_min = min(hi_min, s.hi[mt]);
    }
    s.ev = E_NONE;
    s.lo_min = __builtin_amdgcn_readfirstlane(row16_min_int(lo_min));
    s.hi_max = -__builtin_amdgcn_readfirstlane(row16_min_int(-hi_max));
    s.lo_max = -__builtin_amdgcn_readfirstlane(row16_min_int(-lo_max));
    s.hi_min = __builtin_amdgcn_readfirstlane(row16_min_int(hi_min));
}

// Stores this lane's share of row mt: the normalised output, and for a part
// its (max, sum).
template <int MT>
__device__ __forceinline__ void store_row(const Rows<MT> &s, int mt, float *out, float *ml, int lane) {
    const float l = col4_sum(s.l[mt]);
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
    const int e = s.ev == E_NONE ? 0 : s.ev - X_EXP - P_EXP;
    if (!out) return;
#pragma unroll
    for (int T = 0; T < 4; T++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            f32x4 x;
#pragma unroll
            for (int t = 0; t < 4; t++) x[t] = __builtin_amdgcn_ldexpf(s.o[mt][4 * T + t][r] * inv, e);
            *reinterpret_cast<f32x4 *>(out + 64 * T + 16 * (lane >> 4) + 4 * r) = x;
        }
    if (ml && lane < 16) {
        ml[0] = s.m[mt];
        ml[1] = l;
    }
}

// ---- packed prompts ------------------------------------------------------------

// Row blocks of a sequence of n tokens.
__device__ __forceinline__ int row_blocks(const g3k_paged_args &a, int n, int rows) {
    const int t = rows / a.group;   // tokens per block
    return (n + t - 1) / t;
}

// Block `blk` of the batch: its sequence and rows, the last block of each
// sequence first (the one with the most keys).  False past the last block.
__device__ bool find_block(const g3k_paged_args &a, int blk, int rows, int lane, Unit &u) {
    int before = 0;
    for (int base = 0; base < a.s.num_seqs; base += 64) {
        int first = 0, n = 0;
        if (base + lane < a.s.num_seqs) seq_rows(a.s, base + lane, first, n);
        const int nb = row_blocks(a, n, rows);
        const int upto = wave_scan_int(nb, lane);
        const uint64_t past = __builtin_amdgcn_ballot_w64(blk - before < upto);
        if (past) {
            const int at = __builtin_ctzll(past);
            const int b = base + at;
            const int rb = __shfl(upto, at) - 1 - (blk - before);
            n = __builtin_amdgcn_readfirstlane(__shfl(n, at));
            first = __builtin_amdgcn_readfirstlane(__shfl(first, at));
            const int t = rows / a.group;
            const int tok = __builtin_amdgcn_readfirstlane(rb) * t;
            const int left = n - tok < t ? n - tok : t;
            const int len = __builtin_amdgcn_readfirstlane(seq_len(a.s, b));
            u.b = b;
            u.run = first + tok;
            u.pos = len - n + tok;
            u.first = 0;
            u.count = left * a.group;
            u.kend = u.pos + left > 0 ? u.pos + left : 0;
            u.kbeg = u.pos + 1 - a.window > 0 ? u.pos + 1 - a.window : 0;
            return true;
        }
        before += __shfl(upto, 63);
    }
    return false;
}

// Parts of a block's keys: at least PART_TILES tiles each, at most `most`.
constexpr int PART_TILES = 8;
__device__ __forceinline__ int split_keys(const Unit &u, int most, int part, int &kbeg, int &kend) {
    const int t0 = u.kbeg / BK, n = u.kend > u.kbeg ? (u.kend + BK - 1) / BK - t0 : 0;
    int parts = n / PART_TILES < most ? n / PART_TILES : most;
    if (parts < 1) parts = 1;
    const int per = (n + parts - 1) / parts;
    parts = per > 0 ? (n + per - 1) / per : 1;
    const int b = (t0 + part * per) * BK, e = (t0 + part * per + per) * BK;
    kbeg = b > u.kbeg ? b : u.kbeg;
    kend = e < u.kend ? e : u.kend;
    return parts;
}

template <bool BF16, int MT>
__global__ __launch_bounds__(256, 1) void paged_prefill_kernel(g3k_paged_args a) {
    __shared__ __align__(16) char lds[Lds<BF16>::BYTES];
    __shared__ f32x4 factors[8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = blockIdx.x % a.n_kv_heads, item = blockIdx.x / a.n_kv_heads;
    const int part = item % a.parts, blk = item / a.parts;
    constexpr int ROWS = 64 * MT;
    Unit u;
    if (!find_block(a, blk, ROWS, lane, u)) return;
    int kbeg, kend;
    const int parts = split_keys(u, a.parts, part, kbeg, kend);
    if (part >= parts) return;
    Rows<MT> s;
    const int gs = __builtin_ctz(a.group);
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const int row = (wave * MT + mt) * 16 + (lane & 15);
        const bool live = row < u.count;
        const int tok = row >> gs, h = head * a.group + (row & (a.group - 1));
        const int hi = u.pos + tok + 1;
        s.hi[mt] = live ? min(hi, kend) : INT_MAX;
        s.lo[mt] = live ? max(hi - a.window, kbeg) : 0;
        load_query<MT>(a.q + ((long long)(u.run + tok) * a.n_kv_heads * a.group + h) * D, live, a.qscale, mt, lane, s);
    }
    begin_rows<MT>(s);
    u.kbeg = kbeg;
    u.kend = kend;
    walk<BF16, MT>(a, head, u, lds, factors, wave, lane, s);
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const int row = (wave * MT + mt) * 16 + (lane & 15);
        float *out = nullptr, *ml = nullptr;
        if (row < u.count) {
            if (parts > 1) {
                const long long slot = ((long long)(blk * a.parts + part) * a.n_kv_heads + head) * ROWS + row;
                out = a.part_o + slot * D;
                ml = a.part_ml + slot * 2;
            } else {
                out = a.out + ((long long)(u.run + (row >> gs)) * a.n_kv_heads * a.group + head * a.group +
                               (row & (a.group - 1))) * D;
            }
        }
        store_row<MT>(s, mt, out, ml, lane);
    }
}

// Sums n parts of a row, part i at o + i * stride rows; every lane 4 dims.
// n <= 64; the statistics are one load a lane.
struct Joined {
    f32x4 o;
    float m, l;
};
__device__ __forceinline__ void join_parts(const float *o, const float *ml, long long stride, int n, int lane, Joined &j) {
    for (int base = 0; base < n; base += 64) {
        const int k = n - base < 64 ? n - base : 64;
        float m = M_NONE, l = 0.f;
        if (lane < k) {
            const float *p = ml + (base + lane) * stride * 2;
            m = p[0];
            l = p[1];
        }
        const float top = fmaxf(wave_max(m), j.m);
        const float w = l * fast_exp2(m - top);
        const float keep = fast_exp2(j.m - top);
        j.o *= keep;
        j.l = j.l * keep + wave_sum(w);
        j.m = top;
        for (int i = 0; i < k; i++) {
            const float wi = __shfl(w, i);
            // a part without a visible key has no say, whatever its output
            if (wi != 0.f) j.o += wi * *reinterpret_cast<const f32x4 *>(o + (base + i) * stride * D + 4 * lane);
        }
    }
}

// One wave per row of a block whose keys were split.
template <int MT>
__global__ __launch_bounds__(256) void paged_prefill_merge_kernel(g3k_paged_args a) {
    constexpr int ROWS = 64 * MT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int PER = ROWS / 4;     // workgroups per (block, head)
    const int r4 = blockIdx.x % PER, x = blockIdx.x / PER;
    const int head = x % a.n_kv_heads, blk = x / a.n_kv_heads;
    Unit u;
    if (!find_block(a, blk, ROWS, lane, u)) return;
    int kbeg, kend;
    const int parts = split_keys(u, a.parts, 0, kbeg, kend);
    const int row = r4 * 4 + wave;
    if (parts == 1 || row >= u.count) return;
    const long long slot = ((long long)blk * a.parts * a.n_kv_heads + head) * ROWS + row;
    Joined j = {{0.f, 0.f, 0.f, 0.f}, M_NONE, 0.f};
    join_parts(a.part_o + slot * D, a.part_ml + slot * 2, (long long)a.n_kv_heads * ROWS, parts, lane, j);
    const int gs = __builtin_ctz(a.group);
    float *out = a.out + ((long long)(u.run + (row >> gs)) * a.n_kv_heads * a.group + head * a.group + (row & (a.group - 1))) * D;
    const float inv = j.l > 0.f || j.l != j.l ? 1.0f / j.l : 0.f;
    *reinterpret_cast<f32x4 *>(out + 4 * lane) = j.o * inv;
}

// ---- one query per sequence, shared prefixes ---------------------------------------

// The members [first, end) of group i and the prefix they share; 0 for a
// group of one, whose keys are its own.
__device__ __forceinline__ int group_prefix(const g3k_paged_args &a, int i, int &first, int &end) {
    first = clampi(a.group_start[i], 0, a.s.num_seqs);
    end = clampi(a.group_start[i + 1], first, a.s.num_seqs);
    return end - first < 2 ? 0 : clampi(a.prefix_len[i], 0, a.s.table_stride << a.s.page_shift);
}

// The prefix that sequence b shares, its group's first member in `first`.
__device__ __forceinline__ int seq_prefix(const g3k_paged_args &a, int b, int &first) {
    first = b;
    if (a.n_groups <= 0) return 0;
    int lo = 0, hi = a.n_groups - 1;      // the last group that begins at or before b
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.group_start[mid] <= b) lo = mid;
        else hi = mid - 1;
    }
    int f, e;
    const int p = group_prefix(a, lo, f, e);
    if (b < f || b >= e) return 0;
    first = f;
    return p;
}

__device__ __forceinline__ int tiles_of(int kbeg, int kend) {
    return kend > kbeg ? (kend + BK - 1) / BK - kbeg / BK : 0;
}
// The keys of a prefix that some member may see, and of a sequence beyond it.
__device__ __forceinline__ int prefix_begin(const g3k_paged_args &a, int p) { return p > a.window ? p - a.window : 0; }
__device__ __forceinline__ int tail_begin(const g3k_paged_args &a, int len, int p) {
    const int lo = len - a.window;
    return lo > p ? lo : p;
}

// The work of a decode: per group and 64 MT members' rows, the prefix's keys;
// per sequence, the keys beyond.  Each is cut into chunks of `chunk` tiles so
// that all of them make about a.budget items per KV head, whatever the
// lengths: every wave adds the lengths up for itself.
constexpr int MAX_TILES = G3K_PAGED_MAX_LEN / BK;
template <int ROWS>
__device__ int chunk_tiles(const g3k_paged_args &a, int lane) {
    float total = 0.f;      // rounded: 1e-4 is added below
    int units = 0;
    for (int base = 0; base < a.n_groups; base += 64) {
        float t = 0.f;
        int n = 0;
        if (base + lane < a.n_groups) {
            int f, e;
            const int p = group_prefix(a, base + lane, f, e);
            if (p > 0) {
                n = ((e - f) * a.group + ROWS - 1) / ROWS;
                t = (float)n * (float)tiles_of(prefix_begin(a, p), p);
            }
        }
        total += wave_sum(t);
        units += wave_sum_int(n);
    }
    for (int base = 0; base < a.s.num_seqs; base += 64) {
        float t = 0.f;
        if (base + lane < a.s.num_seqs) {
            int f;
            const int len = seq_len(a.s, base + lane), p = seq_prefix(a, base + lane, f);
            t = (float)tiles_of(tail_begin(a, len, p), len);
        }
        total += wave_sum(t);
    }
    units += a.s.num_seqs;
    const int room = a.budget - units > 1 ? a.budget - units : 1;
    const float c = total * 1.0001f / (float)room + 1.0f;
    return c < (float)a.min_tiles ? a.min_tiles : c < (float)MAX_TILES ? (int)c : MAX_TILES;
}

// Finds chunk `item`: its unit (keys and rows), whether it is a prefix's, and
// how many chunks its unit has.  index: the chunk's number within the unit.
struct Found {
    bool any, prefix;
    int chunks, index;
};
template <int ROWS>
__device__ Found find_chunk(const g3k_paged_args &a, int item, int per, int lane, Unit &u) {
    Found r = {false, false, 0, 0};
    int before = 0;
    for (int base = 0; base < a.n_groups; base += 64) {
        int f = 0, e = 0, p = 0, n = 0, c = 0;
        if (base + lane < a.n_groups) {
            p = group_prefix(a, base + lane, f, e);
            if (p > 0) {
                c = (tiles_of(prefix_begin(a, p), p) + per - 1) / per;
                n = ((e - f) * a.group + ROWS - 1) / ROWS;
            }
        }
        const int upto = wave_scan_int(n * c, lane);
        const uint64_t past = __builtin_amdgcn_ballot_w64(item - before < upto);
        if (past) {
            const int at = __builtin_ctzll(past);
            c = __shfl(c, at);
            n = __shfl(n, at);
            f = __shfl(f, at);
            e = __shfl(e, at);
            p = __shfl(p, at);
            const int k = item - before - (__shfl(upto, at) - n * c);
            const int block = k / c, rows = (e - f) * a.group - block * ROWS;
            r.any = r.prefix = true;
            r.chunks = c;
            r.index = k % c;
            u.b = f;
            u.run = f + block * (ROWS / a.group);
            u.first = 0;
            u.count = rows < ROWS ? rows : ROWS;
            u.pos = 0;
            u.kbeg = prefix_begin(a, p);
            u.kend = p;
            return r;
        }
        before += __shfl(upto, 63);
    }
    for (int base = 0; base < a.s.num_seqs; base += 64) {
        int kb = 0, len = 0, c = 0;
        if (base + lane < a.s.num_seqs) {
            int f;
            len = seq_len(a.s, base + lane);
            kb = tail_begin(a, len, seq_prefix(a, base + lane, f));
            c = (tiles_of(kb, len) + per - 1) / per;
        }
        const int upto = wave_scan_int(c, lane);
        const uint64_t past = __builtin_amdgcn_ballot_w64(item - before < upto);
        if (past) {
            const int at = __builtin_ctzll(past);
            r.any = true;
            r.chunks = __shfl(c, at);
            r.index = item - before - (__shfl(upto, at) - r.chunks);
            u.b = u.run = base + at;
            u.first = 0;
            u.count = a.group;
            u.pos = 0;
            u.kbeg = __shfl(kb, at);
            u.kend = __shfl(len, at);
            return r;
        }
        before += __shfl(upto, 63);
    }
    return r;
}

// Rows of a part: a prefix chunk's ROWS, a tail chunk's group heads.
template <bool BF16, int MT>
__global__ __launch_bounds__(256, 1) void paged_decode_kernel(g3k_paged_args a) {
    __shared__ __align__(16) char lds[Lds<BF16>::BYTES];
    __shared__ f32x4 factors[8];
    constexpr int ROWS = 64 * MT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = blockIdx.x % a.n_kv_heads, item = blockIdx.x / a.n_kv_heads;
    const int per = __builtin_amdgcn_readfirstlane(chunk_tiles<ROWS>(a, lane));
    Unit u;
    Found f = find_chunk<ROWS>(a, item, per, lane, u);
    if (!f.any) return;
    u.b = __builtin_amdgcn_readfirstlane(u.b);
    u.run = __builtin_amdgcn_readfirstlane(u.run);
    u.count = __builtin_amdgcn_readfirstlane(u.count);
    f.chunks = __builtin_amdgcn_readfirstlane(f.chunks);
    f.index = __builtin_amdgcn_readfirstlane(f.index);
    const int t0 = __builtin_amdgcn_readfirstlane(u.kbeg) / BK, kb = (t0 + f.index * per) * BK;
    const int ke = kb + per * BK;
    u.kbeg = max(__builtin_amdgcn_readfirstlane(u.kbeg), kb);
    u.kend = min(__builtin_amdgcn_readfirstlane(u.kend), ke);
    // where the parts of this unit's rows are, for the merge
    int *dir = f.prefix ? a.dir_prefix : a.dir_tail;
    if (f.index == 0 && head == 0 && threadIdx.x == 0) {
        dir[2 * u.run] = item;
        dir[2 * u.run + 1] = f.chunks;
    }
    Rows<MT> s;
    const int gs = __builtin_ctz(a.group);
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const int row = (wave * MT + mt) * 16 + (lane & 15);
        const bool live = row < u.count;
        const int seq = u.run + (row >> gs), h = head * a.group + (row & (a.group - 1));
        const int len = live ? seq_len(a.s, seq) : 0;
        s.hi[mt] = live ? min(len, u.kend) : INT_MAX;
        s.lo[mt] = live ? max(len - a.window, u.kbeg) : 0;
        load_query<MT>(a.q + ((long long)seq * a.n_kv_heads * a.group + h) * D, live, a.qscale, mt, lane, s);
    }
    begin_rows<MT>(s);
    walk<BF16, MT>(a, head, u, lds, factors, wave, lane, s);
    int first;
    const bool whole = !f.prefix && f.chunks == 1 && seq_prefix(a, u.b, first) == 0;
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const int row = (wave * MT + mt) * 16 + (lane & 15);
        float *out = nullptr, *ml = nullptr;
        if (row < u.count) {
            if (whole) {
                out = a.out + ((long long)(u.run + (row >> gs)) * a.n_kv_heads * a.group + head * a.group +
                               (row & (a.group - 1))) * D;
            } else {
                const long long slot = ((long long)item * a.n_kv_heads + head) * a.part_rows + row;
                out = a.part_o + slot * D;
                ml = a.part_ml + slot * 2;
            }
        }
        store_row<MT>(s, mt, out, ml, lane);
    }
}

// One wave per sequence and query head.
template <int MT>
__global__ __launch_bounds__(256) void paged_decode_merge_kernel(g3k_paged_args a) {
    constexpr int ROWS = 64 * MT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int heads = a.n_kv_heads * a.group;
    const long long id = (long long)blockIdx.x * 4 + wave;
    if (id >= (long long)a.s.num_seqs * heads) return;
    const int b = (int)(id / heads), h = (int)(id % heads);
    const int kvh = h / a.group, hg = h % a.group;
    int first;
    const int len = seq_len(a.s, b), p = seq_prefix(a, b, first);
    const int tail = tiles_of(tail_begin(a, len, p), len) > 0;
    // (kept within the parts whatever the directory holds: a batch whose group
    // bounds overlap leaves entries unwritten)
    const int at = tail ? clampi(a.dir_tail[2 * b], 0, a.items - 1) : 0;
    const int chunks = tail ? clampi(a.dir_tail[2 * b + 1], 0, a.items - at) : 0;
    if (p == 0 && chunks == 1) return;        // written by its one chunk
    const long long stride = (long long)a.n_kv_heads * a.part_rows;
    Joined j = {{0.f, 0.f, 0.f, 0.f}, M_NONE, 0.f};
    if (tail) {
        const long long slot = ((long long)at * a.n_kv_heads + kvh) * a.part_rows + hg;
        join_parts(a.part_o + slot * D, a.part_ml + slot * 2, stride, chunks, lane, j);
    }
    if (p > 0) {
        const int row = (b - first) * a.group + hg, lead = first + row / ROWS * (ROWS / a.group);
        const int item = clampi(a.dir_prefix[2 * lead], 0, a.items - 1);
        const long long slot = ((long long)item * a.n_kv_heads + kvh) * a.part_rows + row % ROWS;
        join_parts(a.part_o + slot * D, a.part_ml + slot * 2, stride, clampi(a.dir_prefix[2 * lead + 1], 0, a.items - item), lane, j);
    }
    const float inv = j.l > 0.f || j.l != j.l ? 1.0f / j.l : 0.f;
    *reinterpret_cast<f32x4 *>(a.out + id * D + 4 * lane) = j.o * inv;
}

}  // namespace

extern "C" int g3k_paged_prefill(const g3k_paged_args *a, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    const long long wgs = (long long)a->items * a->parts * a->n_kv_heads;
    const long long merges = (long long)a->items * a->n_kv_heads * 16 * a->blocks;
    if (wgs > INT_MAX || merges > INT_MAX) return (int)hipErrorInvalidValue;
    const dim3 grid((unsigned)wgs), merge((unsigned)merges);
    {
        if (a->bf16) hipLaunchKernelGGL((paged_prefill_kernel<true, 1>), grid, dim3(256), 0, st, *a);
        else hipLaunchKernelGGL((paged_prefill_kernel<false, 1>), grid, dim3(256), 0, st, *a);
        if (a->parts > 1) hipLaunchKernelGGL(paged_prefill_merge_kernel<1>, merge, dim3(256), 0, st, *a);
    }
    return (int)hipGetLastError();
}

extern "C" int g3k_paged_decode(const g3k_paged_args *a, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    const long long wgs = (long long)a->items * a->n_kv_heads;
    const long long merges = ((long long)a->s.num_seqs * a->n_kv_heads * a->group + 3) / 4;
    if (wgs > INT_MAX || merges > INT_MAX) return (int)hipErrorInvalidValue;
    const dim3 grid((unsigned)wgs), merge((unsigned)merges);
    {
        if (a->bf16) hipLaunchKernelGGL((paged_decode_kernel<true, 1>), grid, dim3(256), 0, st, *a);
        else hipLaunchKernelGGL((paged_decode_kernel<false, 1>), grid, dim3(256), 0, st, *a);
        hipLaunchKernelGGL(paged_decode_merge_kernel<1>, merge, dim3(256), 0, st, *a);
    }
    return (int)hipGetLastError();
}
