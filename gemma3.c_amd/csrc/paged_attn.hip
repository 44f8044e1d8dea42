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
// One workgroup = 8 waves (4 for short prompts, with twice the keys a wave to
// convert) = one KV head x 128 query rows (a row is one query
// head of one token; the heads of a group share the keys); each wave owns 16
// rows over the full head dim (Q hi / lo 64 VGPRs, O^T 64) and walks 32-key
// tiles that the waves load and convert together:
//   S^T[key][row] = K . Q^T,  O^T[dim][row] += V^T . P^T,
// both v_mfma_f32_16x16x32_f16.  In the 16x16 accumulator lane l holds column
// (row) l % 16, so a row's softmax state lives in the lanes l % 16 + 16 g.
// 32 rows a wave would halve the LDS reads a row, but their O^T and Q leave no
// registers for the tiles in flight (they spilled).
//
// What bounds it: packed fp32 prompts of 8192 tokens (8 heads over 4) take 430
// us, 120 GFLOP and 378 on the matrix units, 66% of the rate a large fp16
// product of the library reaches; matrix units busy 42% of the cycles, vector
// units 34%, LDS 42%, at 2.0 GHz.  bf16 chunks: 285 us, 313 TFLOP/s, twice that
// on the matrix units.  A tile takes 6400 cycles (bf16 5500): 2700 (2000) on
// scores and values, 3300 (2900) on softmax and the next tiles' conversion, in
// which a SIMD's two waves are opposite.  With every tile already in the cache
// it is 3% quicker.
//
// LDS holds a tile as MFMA A operands in lane order (1 KiB each, so every
// read is one conflict-free ds_read_b128): K [2 key blocks][8 dim steps], V
// [16 dim blocks], each hi then lo.  Wave w brings keys 16 (w / 4) + 4 g.. of
// g = w % 4, one coalesced row per load.  These are the keys lane group g of
// the S^T registers holds, so P goes from the S^T registers to the
// P.V operand without a shuffle, and one scale per wave and tile is one
// factor per lane group: K's on the scores, V's on P.  A V lane holds 4 dims
// of the 8 keys, which are whole operand lanes of the four dim blocks
// {64 T + 4 c + t}: the transposition is register naming.  K lanes write half
// an operand lane (4 dims) each, at a position XORed by the dim step, so the
// 8-byte stores spread over the banks.
#include <hip/hip_runtime.h>
#include <limits.h>

#include <type_traits>

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
constexpr int NOTES = 8;                    // of a tile: one per run and lane group; behind both tiles', unused ones
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

// Keeps the matrix operands' LDS reads and their MFMAs in the written order
// (one step ahead), so that they take few registers; everything else moves
// freely across.  Scheduler mask: VALU, SALU, vector memory, LDS writes.
#define KEEP_OPERANDS() __builtin_amdgcn_sched_barrier(0x2 | 0x4 | 0x10 | 0x20 | 0x40 | 0x200)

__device__ __forceinline__ half2v cvt2(float a, float b) { return __builtin_convertvector((f32x2){a, b}, half2v); }

// The larger of two, NaN if either is (v_maximum3_f32: no canonicalising moves
// before it, as before v_max_f32), and so over a row's lanes and the wave's.
__device__ __forceinline__ float top(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float col4_top(float v) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = top(__uint_as_float(x[0]), __uint_as_float(x[1]));
    const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return top(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
__device__ __forceinline__ float wave_top(float v) {
    v = top(v, dpp<0xB1>(v));      // within quads, their pairs, eights, sixteens
    v = top(v, dpp<0x4E>(v));
    v = top(v, dpp<0x141>(v));
    v = top(v, dpp<0x140>(v));
    return col4_top(v);
}

// The wave's largest of values >= 0, as bits: so ordered, NaN above all.
__device__ __forceinline__ int wave_top_bits(float v) {
    unsigned x = __float_as_uint(v);
    const auto up = [&](unsigned y) { x = x > y ? x : y; };
    up(__builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true));     // row_shr:1, 2, 4, 8
    up(__builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true));
    up(__builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true));
    up(__builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true));
    up(__builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false));    // row_bcast:15 to rows 1 and 3
    up(__builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false));    // row_bcast:31 to rows 2 and 3
    return __builtin_amdgcn_readlane((int)x, 63);
}

// The power-of-two exponent of a block whose largest magnitude has these bits:
// it is below 2^exponent.  A block of zeros, or of values below 2^-100, counts
// as 2^-100; one with an infinity or NaN as 2^129 (X_EXP - 129 is still the
// exponent of a normal number).
constexpr int NOT_FINITE = 0x7f800000;
__device__ __forceinline__ int block_exponent(int bits) { return max((bits >> 23) - 126, -100); }
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// x s as hi + lo, two values at a time.
__device__ __forceinline__ void split2(float a, float b, float s, half2v &hi, half2v &lo) {
    hi = cvt2(a * s, b * s);
    lo.x = (_Float16)__builtin_fmaf(a, s, -(float)hi.x);
    lo.y = (_Float16)__builtin_fmaf(b, s, -(float)hi.y);
}

// What a workgroup attends: the rows of a run of tokens over keys [kbeg, kend)
// of table row b.
struct Unit {
    int b, kbeg, kend;
    int count;             // rows (of the group's heads)
    int run;               // prefill: packed row of the run's first token; decode: the run's first sequence
    int pos;               // prefill: position of that token
};

// ---- the tile walk -----------------------------------------------------------

template <bool BF16>
struct Lds {
    static constexpr int PL = BF16 ? 1 : 2;            // planes
    static constexpr int K_BYTES = 2 * 8 * PL * 1024;  // [key block][dim step][plane] operands
    static constexpr int V_BYTES = 16 * PL * 1024;     // [dim block][plane]
    static constexpr int BYTES = 2 * (K_BYTES + V_BYTES);
};

// Rows of one matrix in flight: this wave's share of a tile's 32 keys, 4 dims
// a lane.  Of NW waves, wave w brings lane group g = w % 4's keys: with 4 both
// runs 4 g.. and 16 + 4 g.., with 8 the run 16 (w / 4) + 4 g...
template <bool BF16, int NW>
struct Raw {
    static constexpr int RUNS = 8 / NW;
    typename std::conditional<BF16, u32x2, f32x4>::type x[4 * RUNS];
    __device__ __forceinline__ f32x4 get(int i) const {
        if constexpr (BF16) {
            const u32x2 u = x[i];
            return (f32x4){__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                           __uint_as_float(u.y & 0xffff0000u)};
        } else {
            return x[i];
        }
    }
    __device__ __forceinline__ void set(int i, unsigned bits) {
        if constexpr (BF16) x[i] = (u32x2){bits, bits};
        else x[i] = (f32x4){__uint_as_float(bits), __uint_as_float(bits), __uint_as_float(bits), __uint_as_float(bits)};
    }
};

__device__ const float zero_row[D] = {};

// Pages and zero_row as what they are, global memory: through a generic
// pointer their loads would count as LDS accesses too, and every wait for LDS,
// barriers included, would be one for the rows in flight (packed prompts of
// 8192 tokens: 514 us against 462).
typedef const G3K_GLOBAL char *gbytes;
template <class T>
__device__ __forceinline__ T load_global(gbytes p) { return *reinterpret_cast<const G3K_GLOBAL T *>(p); }
__device__ __forceinline__ gbytes global_bytes(const void *p) { return (gbytes)p; }

// Where the rows of a walk are.  Looks pages up along it: 64 table entries in
// a register, the next 64 on their way, so that a tile's lookup waits for no
// memory.  A tile's entries never straddle two such runs (a tile is one
// entry, or two from an even one).
template <bool BF16, int NW>
struct Finder {
    static constexpr int RUNS = 8 / NW, ROW = D * (BF16 ? 2 : 4);
    // A wave's share of a tile: byte offset of each run's first row from the
    // head's first page, this lane's offsets of its rows from there, and which
    // runs have no page.
    struct Place {
        long long off[RUNS];
        unsigned row[4 * RUNS];
        int bad, none;
    };
    const int *table;
    int shift, mask, last, pages, kbeg, kend;     // last: entry of the walk
    unsigned stride;                              // elements between pages
    int base, now, next;
    gbytes zeros;

    __device__ __forceinline__ void begin(const g3k_paged_args &a, const Unit &u, int lane) {
        table = a.s.page_table + (long long)u.b * a.s.table_stride;
        shift = a.s.page_shift;
        mask = (1 << shift) - 1;
        last = (u.kend - 1) >> shift;
        pages = a.num_pages;
        stride = (unsigned)a.page_stride;
        kbeg = u.kbeg;
        kend = u.kend;
        base = (kbeg >> shift) & ~63;
        zeros = global_bytes(zero_row);
        G3K_RECOMPUTE_S(zeros);
        now = table[clampi(base + lane, 0, last)];
        next = table[clampi(base + 64 + lane, 0, last)];
    }
    __device__ __forceinline__ Place place(int tile, int wave, int lane) {
        Place p;
        p.bad = p.none = 0;
        const int j0 = tile * BK;
        if ((j0 >> shift) >= base + 64) {
            base += 64;
            now = next;
            next = table[clampi(base + 64 + lane, 0, last)];
        }
#pragma unroll
        for (int r = 0; r < RUNS; r++) {
            const int j = j0 + 16 * (NW == 4 ? r : wave >> 2);
            // (a run wholly outside the keys looks its nearest key's page up)
            const int e = clampi(j, kbeg & ~15, kend - 1) >> shift;
            const unsigned page = __builtin_amdgcn_readlane(now, e - base);
            // Keys outside [kbeg, kend) take the nearest row of their run
            // inside, so nothing else is read; their scores are masked.  A page
            // outside the pool is never followed, and neither is a run without
            // a key: the rows are zeros.
            const int from = max(kbeg - j, 0), to = min(kend - 1 - j, 15);
            const bool bad = page >= (unsigned)pages, none = bad || from > to;
            const int lo = none ? 0 : from, hi = none ? 0 : to;
            if (bad) p.bad |= 1 << r;
            if (none) p.none |= 1 << r;
            p.off[r] = (long long)(((unsigned long long)page * stride + (unsigned)((j & mask) * D)) * (BF16 ? 2 : 4));
#pragma unroll
            for (int i = 0; i < 4; i++)
                p.row[4 * r + i] = (unsigned)min(max(4 * (wave & 3) + i, lo), hi) * ROW + (unsigned)lane * (ROW / 64);
        }
        return p;
    }
    __device__ __forceinline__ void fetch(gbytes matrix, const Place &p, Raw<BF16, NW> &raw) const {
        using T = typename std::conditional<BF16, u32x2, f32x4>::type;
#pragma unroll
        for (int r = 0; r < RUNS; r++) {
            const gbytes rows = (p.none >> r) & 1 ? zeros : matrix + p.off[r];
#pragma unroll
            for (int i = 0; i < 4; i++) raw.x[4 * r + i] = load_global<T>(rows + p.row[4 * r + i]);
        }
    }
};

// The largest magnitude of this lane's share of the rows in flight.
template <bool BF16, int NW>
__device__ __forceinline__ float rows_max(const Raw<BF16, NW> &raw) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 4 * Raw<BF16, NW>::RUNS; i++) {
        const f32x4 x = raw.get(i);
        m = top(top(m, fabsf(x.x)), fabsf(x.y));
        m = top(top(m, fabsf(x.z)), fabsf(x.w));
    }
    return m;
}

// The largest finite magnitude (its bits) of this wave's rows in flight, where
// some hold an infinity or a NaN (seldom any): those rows, one bit each in
// `spoiled`, are left out of the exponent, which is their neighbours' too.  K's
// become NaN, and so their scores, which are masked for the rows that do not
// see them.  V's become zeros, since a value that is not finite times p = 0 is
// NaN in every row of the product; a row that sees the key is made NaN instead.
// (Looking for them costs 1%.)
template <bool KEYS, bool BF16, int NW>
__device__ __forceinline__ int settle(Raw<BF16, NW> &raw, int &spoiled) {
    spoiled = 0;
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 4 * Raw<BF16, NW>::RUNS; i++) {
        const f32x4 x = raw.get(i);
        const float y = top(top(fabsf(x.x), fabsf(x.y)), top(fabsf(x.z), fabsf(x.w)));
        if (__builtin_amdgcn_ballot_w64(!(y < INFINITY))) {
            spoiled |= 1 << i;
            raw.set(i, KEYS ? BF16 ? 0x7fc07fc0u : 0x7fc00000u : 0u);
        } else {
            most = top(most, y);
        }
    }
    return wave_top_bits(most);
}

// K's rows (exponent e over the wave) as operands: lane holds dims 4 lane.. =
// half (lane & 1) of operand lane group (lane >> 1) & 3 of dim step lane >> 3.
// factors[run][group]: what the scores of these keys are multiplied by, and
// their additive mask (lane 0's; the others write where nothing is read, which
// saves a branch).
template <bool BF16, int NW>
__device__ __forceinline__ void store_k(const Raw<BF16, NW> &raw, int e, int bad, char *buf, f32x2 *factors, int wave, int lane) {
    using L = Lds<BF16>;
    const float sc = pow2(X_EXP - e);
    char *kd = buf + (lane >> 3) * (L::PL * 1024) + ((lane >> 1) & 3) * 256 + (lane & 1) * 8;
    const int f = (lane >> 1) & 15;
#pragma unroll
    for (int r = 0; r < Raw<BF16, NW>::RUNS; r++) {
        const int c = NW == 4 ? r : wave >> 2;
        factors[lane ? 2 * NOTES + lane : 4 * c + (wave & 3)] = (f32x2){pow2(e - X_EXP), (bad >> r) & 1 ? -INFINITY : 0.f};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f32x4 x = raw.get(4 * r + i);
            char *d = kd + c * (8 * L::PL * 1024) + (((4 * (wave & 3) + i) ^ f) << 4);
            half4v h, l;
            if constexpr (BF16) {
                h.xy = cvt2(x.x * sc, x.y * sc);
                h.zw = cvt2(x.z * sc, x.w * sc);
            } else {
                half2v p, q;
                split2(x.x, x.y, sc, p, q);
                h.xy = p;
                l.xy = q;
                split2(x.z, x.w, sc, p, q);
                h.zw = p;
                l.zw = q;
                *reinterpret_cast<half4v *>(d + 1024) = l;
            }
            *reinterpret_cast<half4v *>(d) = h;
        }
    }
}

// V's rows as operands: lane holds dims 4 lane + t of operand lane lane & 15 of
// group g of dim blocks 4 (lane >> 4) + t, its keys 4 c.. of the operand's 8.
// exps[run][group]: the exponent of these keys in 12 bits, above them one bit
// for each spoiled key.
template <bool BF16, int NW>
__device__ __forceinline__ void store_v(const Raw<BF16, NW> &raw, int e, int spoiled, char *buf, int *exps, int wave, int lane) {
    using L = Lds<BF16>;
    constexpr int N = 4 * Raw<BF16, NW>::RUNS;
    typedef _Float16 Keys __attribute__((ext_vector_type(N)));
    const float sc = pow2(X_EXP - e);
    const int c = NW == 4 ? 0 : wave >> 2;
    // (with 4 waves lane 1 has the second run's)
    const int run = NW == 4 ? lane & 1 : 0;
    exps[lane < 8 / NW ? 4 * (c + run) + (wave & 3) : 2 * NOTES + lane] = e + ((spoiled >> 4 * run & 15) << 12);
    char *vd = buf + (lane >> 4) * (4 * L::PL * 1024) + (wave & 3) * 256 + (lane & 15) * 16 + c * 8;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        Keys h, l;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float x = raw.get(i)[t], y = raw.get(i + 1)[t];
            half2v hh, ll;
            if constexpr (BF16) {
                hh = cvt2(x * sc, y * sc);
            } else {
                split2(x, y, sc, hh, ll);
                l[i] = ll.x;
                l[i + 1] = ll.y;
            }
            h[i] = hh.x;
            h[i + 1] = hh.y;
        }
        *reinterpret_cast<Keys *>(vd + t * (L::PL * 1024)) = h;
        if constexpr (!BF16) *reinterpret_cast<Keys *>(vd + t * (L::PL * 1024) + 1024) = l;
    }
}

// The rows of a wave: queries in registers, running softmax state, O^T.
struct Rows {
    half8 qh[8], ql[8];
    f32x4 o[16];
    float factor, m, l;               // l: this lane's keys only
    int lo, hi;                       // the keys this lane's row sees
    int lo_max, hi_min;               // over the wave's rows: tiles between them need no mask
    int ev;                           // O^T's exponent: o = true o * 2^(X_EXP + P_EXP - ev), unnormalised
};

// A row's query: this lane group's 8 of every 32 dims, and their split planes.
struct Query {
    f32x4 x[8][2];
    __device__ __forceinline__ void load(const float *q, bool live, int lane) {
#pragma unroll
        for (int kk = 0; kk < 8; kk++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const f32x4 z = {0.f, 0.f, 0.f, 0.f};
                x[kk][i] = live ? *reinterpret_cast<const f32x4 *>(q + 32 * kk + 8 * (lane >> 4) + 4 * i) : z;
            }
    }
    __device__ __forceinline__ void split(float qscale, Rows &s) const {
        float m = 0.f;
#pragma unroll
        for (int kk = 0; kk < 8; kk++)
#pragma unroll
            for (int i = 0; i < 8; i++) m = top(m, fabsf(x[kk][i >> 2][i & 3]));
        const int e = block_exponent(__float_as_int(col4_top(m)));
        const float sc = pow2(X_EXP - e);
        s.factor = __builtin_amdgcn_ldexpf(qscale, e - X_EXP);
#pragma unroll
        for (int kk = 0; kk < 8; kk++)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                half2v h, l;
                split2(x[kk][i >> 2][i & 3], x[kk][i >> 2][(i & 3) + 1], sc, h, l);
                s.qh[kk][i] = h.x;
                s.qh[kk][i + 1] = h.y;
                s.ql[kk][i] = l.x;
                s.ql[kk][i + 1] = l.y;
            }
    }
};

// S^T of a tile.
template <bool BF16>
__device__ __forceinline__ void tile_scores(const char *buf, int lane, const Rows &s, f32x4 (&sc)[2]) {
    using L = Lds<BF16>;
    const int g = lane >> 4, c = lane & 15;
    f32x4 sx[2];                  // the products with a lo plane: four sums, so that
    sc[0] = sc[1] = sx[0] = sx[1] = (f32x4){0.f, 0.f, 0.f, 0.f};   // none waits for its last MFMA
    half8 kh[2][2], kl[2][2];     // operands of this dim step and the next
    const auto read = [&](int kk) {
        const char *kp = buf + kk * (L::PL * 1024) + g * 256 + ((c ^ ((4 * kk + g) & 15)) << 4);
#pragma unroll
        for (int kt = 0; kt < 2; kt++) {
            kh[kk & 1][kt] = *reinterpret_cast<const half8 *>(kp + kt * (8 * L::PL * 1024));
            if constexpr (!BF16) kl[kk & 1][kt] = *reinterpret_cast<const half8 *>(kp + kt * (8 * L::PL * 1024) + 1024);
        }
    };
    read(0);
#pragma unroll
    for (int kk = 0; kk < 8; kk++) {
        const int x = kk & 1;
        if (kk < 7) read(kk + 1);
        sc[0] = mfma(kh[x][0], s.qh[kk], sc[0]);
        sx[0] = mfma(kh[x][0], s.ql[kk], sx[0]);
        sx[1] = mfma(kh[x][1], s.ql[kk], sx[1]);
        sc[1] = mfma(kh[x][1], s.qh[kk], sc[1]);
        if constexpr (!BF16) {
            sx[0] = mfma(kl[x][0], s.qh[kk], sx[0]);
            sx[1] = mfma(kl[x][1], s.qh[kk], sx[1]);
        }
        KEEP_OPERANDS();
    }
    sc[0] += sx[0];
    sc[1] += sx[1];
}

// Scores to probabilities (in place), the running max and sum, and O^T's
// rescaling, which is rare: a row's max moves only when a score outgrows it by
// 2^LAZY.  fac[run]: the factor and mask of this lane group's keys.
__device__ __forceinline__ void tile_softmax(const f32x2 (&fac)[2], int tile, int lane, Rows &s, f32x4 (&sc)[2]) {
    const int j0 = tile * BK;
    const bool ragged = j0 < s.lo_max || j0 + BK > s.hi_min;
    float t = M_NONE;
#pragma unroll
    for (int kt = 0; kt < 2; kt++) {
        const float f = s.factor * fac[kt].x;
#pragma unroll
        for (int r = 0; r < 4; r++) sc[kt][r] = __builtin_fmaf(sc[kt][r], f, fac[kt].y);
    }
    if (ragged) {
        G3K_RECOMPUTE(lane);      // (what follows is not done ahead of the branch)
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int j = j0 + 16 * kt + 4 * (lane >> 4) + r;
                if (j < s.lo || j >= s.hi) sc[kt][r] = -INFINITY;
            }
    }
#pragma unroll
    for (int kt = 0; kt < 2; kt++)
#pragma unroll
        for (int r = 0; r < 4; r++) t = top(t, sc[kt][r]);
    t = col4_top(t);
    const bool up = t > s.m + LAZY;
    if (__builtin_amdgcn_ballot_w64(up)) {
        const float m = up ? t : s.m;
        const float keep = fast_exp2(s.m - m);
        s.m = m;
        s.l *= keep;
#pragma unroll
        for (int d = 0; d < 16; d++) s.o[d] *= keep;
    }
#pragma unroll
    for (int kt = 0; kt < 2; kt++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            sc[kt][r] = fast_exp2(sc[kt][r] - s.m);
            s.l += sc[kt][r];
        }
}

// P of a tile as the operand of P.V, scaled by its keys' V exponent against
// O^T's.  The one O^T is held at is two bits above what the first tile has, so
// ordinary tiles do not move it.
__device__ __forceinline__ int exponent_of(int packed) { return (int)((unsigned)packed << 20) >> 20; }
__device__ __forceinline__ void split_p(const f32x4 (&p)[2], const int *exps, int tile, int lane, Rows &s, half8 &ph, half8 &pl) {
    const int mine[2] = {exps[lane >> 4], exps[4 + (lane >> 4)]};
    int most = exps[0];
#pragma unroll
    for (int i = 1; i < 8; i++) most = max(most, exps[i]);
    int up = __builtin_amdgcn_readfirstlane(most);
    if (up > s.ev) {
        if (up >= 1 << 11) {         // keys are spoiled
            G3K_RECOMPUTE(lane);
            G3K_RECOMPUTE(exps);
            most = exponent_of(exps[0]);
#pragma unroll
            for (int i = 1; i < 8; i++) most = max(most, exponent_of(exps[i]));
            up = __builtin_amdgcn_readfirstlane(most);
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int j = tile * BK + 16 * kt + 4 * (lane >> 4) + r;
                    if (((mine[kt] - exponent_of(mine[kt])) >> (12 + r) & 1) && j >= s.lo && j < s.hi) s.l = NAN;
                }
        }
        if (up > s.ev) {
            const float down = s.ev == E_NONE ? 0.f : __builtin_amdgcn_ldexpf(1.0f, s.ev - up - 2);
            s.ev = up + 2;
#pragma unroll
            for (int d = 0; d < 16; d++) s.o[d] *= down;
        }
    }
#pragma unroll
    for (int kt = 0; kt < 2; kt++) {
        const float f = __builtin_amdgcn_ldexpf(1.0f, P_EXP + exponent_of(mine[kt]) - s.ev);
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
            half2v h, l;
            split2(p[kt][r], p[kt][r + 1], f, h, l);
            ph[4 * kt + r] = h.x;
            ph[4 * kt + r + 1] = h.y;
            pl[4 * kt + r] = l.x;
            pl[4 * kt + r + 1] = l.y;
        }
    }
}

// O^T += V^T P^T of a tile.
template <bool BF16>
__device__ __forceinline__ void tile_values(const char *buf, int lane, half8 ph, half8 pl, Rows &s) {
    using L = Lds<BF16>;
    const char *vp = buf + lane * 16;
    // a step takes hi.hi of one dim block, hi.lo of the last and lo.hi of the
    // one before: no sum waits for its last MFMA
    half8 vh[4], vl[3];
    const auto read_hi = [&](int d) { vh[d & 3] = *reinterpret_cast<const half8 *>(vp + d * (L::PL * 1024)); };
    read_hi(0);
    read_hi(1);
#pragma unroll
    for (int d = 0; d < 18; d++) {
        if (d < 14) read_hi(d + 2);
        if constexpr (!BF16) {
            if (d < 16) vl[d % 3] = *reinterpret_cast<const half8 *>(vp + d * (L::PL * 1024) + 1024);
        }
        if (d < 16) s.o[d] = mfma(vh[d & 3], ph, s.o[d]);
        if (d > 0 && d < 17) s.o[d - 1] = mfma(vh[(d - 1) & 3], pl, s.o[d - 1]);
        if constexpr (!BF16) {
            if (d > 1) s.o[d - 2] = mfma(vl[(d - 2) % 3], ph, s.o[d - 2]);
        }
        KEEP_OPERANDS();
    }
}

// The walk of a workgroup over its unit's tiles, counted from 0 here.  A step
// is a phase on the matrix units, M(i): scores of tile i + 1, values of tile
// i; and one on the vector units, V(i): softmax of tile i + 1, this wave's
// rows of later tiles split and stored (and the next ones fetched).  With 8
// waves, waves w and w + 4 share a SIMD; the second four run one phase later,
// so that one is in M while the other is in V, and store one tile further
// ahead (`lead`).  Tile i + 2 of K goes where tile i was, i + 1 of V where
// i - 1 was, both at least a phase after their last read and before their
// first; what V(i) needs of the factors is read in M(i), before others write
// them.  q: the query of this lane's row, if it is live.
template <bool BF16, int NW>
__device__ __forceinline__ void walk(const g3k_paged_args &a, int head, const Unit &u, char *lds, f32x2 *factors, int *exps, int wave,
                                     int lane, const float *q, bool live, Rows &s) {
    using L = Lds<BF16>;
    const int t0 = u.kbeg / BK, n = u.kend > u.kbeg ? (u.kend + BK - 1) / BK - t0 : 0;
    if (n <= 0) return;
    char *kbuf = lds, *vbuf = lds + 2 * L::K_BYTES;
    const long long head_off = ((long long)head << a.s.page_shift) * D * (BF16 ? 2 : 4);
    const gbytes kb = global_bytes(a.k) + head_off, vb = global_bytes(a.v) + head_off;
    Finder<BF16, NW> find;
    // the pages, the query and the first rows are asked for before any is used
    // (9 short prompts 21.7 us; 0.7 more with the query settled first)
    find.begin(a, u, lane);
    Query query;
    query.load(q, live, lane);
    Raw<BF16, NW> rk, rv;
    // tiles in flight; past the end nothing is fetched, and what is stored again
    // is not read (packed fp32 8192 tokens 432 us; the last tile fetched again 446)
    int ik = 0, iv = 0;
    auto pk = find.place(t0, wave, lane), pv = pk;
    find.fetch(kb, pk, rk);
    find.fetch(vb, pv, rv);
    query.split(a.qscale, s);
    // K's next tile has been looked up when V's is fetched
    const auto next_k = [&](int e) {
        store_k<BF16, NW>(rk, e, pk.bad, kbuf + (ik & 1) * L::K_BYTES, factors + 8 * (ik & 1), wave, lane);
        ik++;
        pv = pk;
        if (ik < n) {
            pk = find.place(t0 + ik, wave, lane);
            find.fetch(kb, pk, rk);
        }
    };
    const auto next_v = [&](int e, int spoiled) {
        store_v<BF16, NW>(rv, e, spoiled, vbuf + (iv & 1) * L::V_BYTES, exps + 8 * (iv & 1), wave, lane);
        iv++;
        if (iv < n) find.fetch(vb, pv, rv);
    };
    const int lead = NW == 8 ? wave >> 2 : 0;
    int spoiled;
    next_k(block_exponent(settle<true>(rk, spoiled)));
    if (lead) {
        pv = pk;
        const int ev = block_exponent(settle<false>(rv, spoiled));
        next_v(ev, spoiled);
        next_k(block_exponent(settle<true>(rk, spoiled)));
    }
    // only LDS has to have arrived at these barriers: 63 vector memory
    // operations may stay in flight
    G3K_WAIT_BARRIER(63);
    if (lead) G3K_WAIT_BARRIER(63);
    f32x4 p[2];             // tile i's scores, then probabilities
    half8 ph, pl;
    for (int i = 0; i < n; i++) {
        const int t = t0 + i, x = i & 1;
        G3K_RECOMPUTE(lane);
        // M(i - 1)
        f32x4 sc[2];
        const f32x2 *f = factors + 8 * x + (lane >> 4);
        const f32x2 fac[2] = {f[0], f[4]};
        tile_scores<BF16>(kbuf + x * L::K_BYTES, lane, s, sc);
        if (i > 0) {
            split_p(p, exps + 8 * (x ^ 1), t - 1, lane, s, ph, pl);
            tile_values<BF16>(vbuf + (x ^ 1) * L::V_BYTES, lane, ph, pl, s);
        }
        p[0] = sc[0];
        p[1] = sc[1];
        if (NW == 8) G3K_WAIT_BARRIER(63);
        // V(i - 1)
        // (three chains of cross-lane steps side by side)
        int mk = wave_top_bits(rows_max<BF16, NW>(rk)), mv = wave_top_bits(rows_max<BF16, NW>(rv));
        spoiled = 0;
        tile_softmax(fac, t, lane, s, p);
        if (max(mk, mv) >= NOT_FINITE) {
            mk = settle<true>(rk, spoiled);
            mv = settle<false>(rv, spoiled);
        }
        next_k(block_exponent(mk));
        next_v(block_exponent(mv), spoiled);
        G3K_WAIT_BARRIER(63);
    }
    split_p(p, exps + 8 * ((n - 1) & 1), t0 + n - 1, lane, s, ph, pl);
    tile_values<BF16>(vbuf + ((n - 1) & 1) * L::V_BYTES, lane, ph, pl, s);
    // the second four are a phase behind: one barrier more before, one less after
    if (NW == 8 && !lead) G3K_WAIT_BARRIER(63);
}

// Row state before the walk, from the keys each lane's row sees: [lo, hi),
// or [0, INT_MAX) for a lane without a row.
__device__ __forceinline__ void begin_rows(Rows &s) {
    s.m = M_NONE;
    s.l = 0.f;
#pragma unroll
    for (int d = 0; d < 16; d++) s.o[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    s.ev = E_NONE;
    const bool row = s.hi != INT_MAX;
    s.lo_max = -__builtin_amdgcn_readfirstlane(row16_min_int(row ? -s.lo : 0));
    s.hi_min = __builtin_amdgcn_readfirstlane(row16_min_int(row ? s.hi : INT_MAX));
}

// Stores this lane's share of its row (if it has one): the normalised output,
// and for a part its (max, sum).
__device__ __forceinline__ void store_row(const Rows &s, float *out, float *ml, int lane) {
    const float l = col4_sum(s.l);
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
    const int e = s.ev == E_NONE ? 0 : s.ev - X_EXP - P_EXP;
    if (!out) return;
#pragma unroll
    for (int T = 0; T < 4; T++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            f32x4 x;
#pragma unroll
            for (int t = 0; t < 4; t++) x[t] = __builtin_amdgcn_ldexpf(s.o[4 * T + t][r] * inv, e);
            *reinterpret_cast<f32x4 *>(out + 64 * T + 16 * (lane >> 4) + 4 * r) = x;
        }
    if (ml && lane < 16) {
        ml[0] = s.m;
        ml[1] = l;
    }
}

// ---- packed prompts ------------------------------------------------------------

// A sequence's new tokens as blocks of T tokens (ROWS rows of a head group).
struct Prompt {
    int first, n, pos, blocks;     // packed row, tokens, position of the first, blocks
    bool all;                      // no block's window leaves keys out
    __device__ __forceinline__ int kend(int rb, int T) const {
        const int e = pos + min((rb + 1) * T, n);
        return e > 0 ? e : 0;
    }
    // tiles of the block with the most, or (behind a window) at most that many
    __device__ __forceinline__ int most_tiles(const g3k_paged_args &a, int T) const {
        const int whole = (max(pos + n, 0) + BK - 1) / BK;
        return all ? whole : min(whole, (a.window + T) / BK + 2);
    }
    // the first block with x tiles or more (`blocks`: none); a block's keys end
    // with it
    __device__ __forceinline__ int first_of(int x, int T) const {
        const int y = (x - 1) * BK - pos;
        return x <= 0 || y < 0 ? 0 : y >= n ? blocks : y >> __builtin_ctz(T);      // (T is a power of two)
    }
    // the first with more than p chunks of c tiles (or an earlier one, behind a
    // window)
    __device__ __forceinline__ int first_with(int p, int c, int T) const { return p == 0 || !all ? 0 : first_of(p * c + 1, T); }
    __device__ __forceinline__ int chunks(const g3k_paged_args &a, int c, int T) const {
        const int t = most_tiles(a, T);
        return t > 0 ? (t + c - 1) / c : 1;
    }
    __device__ __forceinline__ int items(const g3k_paged_args &a, int c, int T) const {
        const int k = chunks(a, c, T);
        if (!all || k == 1) return blocks * k;
        int sum = 0;
        for (int p = 0; p < k; p++) sum += blocks - first_with(p, c, T);
        return sum;
    }
};

__device__ __forceinline__ Prompt prompt_of(const g3k_paged_args &a, int b, int T) {
    Prompt p = {0, 0, 0, 0, true};
    if (b >= a.s.num_seqs) return p;
    seq_rows(a.s, b, p.first, p.n);
    const int len = seq_len(a.s, b);
    p.pos = len - p.n;
    p.blocks = (p.n + T - 1) >> __builtin_ctz(T);
    p.all = a.window >= len;
    return p;
}

constexpr int MAX_TILES = G3K_PAGED_MAX_LEN / BK;
constexpr float LONG_TILES = 48.f;

// Tiles per chunk: the longest blocks' keys are cut so that the batch is about
// a.budget items per KV head, or twice as many, whatever the lengths.  Every
// wave adds the lengths up for itself (a causal block has keys up to its last
// token).  Without a budget nothing is cut.
__device__ int prompt_chunk(const g3k_paged_args &a, int T, int lane) {
    if (a.budget <= 0) return MAX_TILES;
    float total = 0.f;      // an upper estimate
    for (int base = 0; base < a.s.num_seqs; base += 64) {
        const Prompt p = prompt_of(a, base + lane, T);
        float t = 0.f;
        if (p.blocks > 0) {
            const float n = (float)p.blocks;
            t = p.all ? n * ((float)max(p.pos, 0) * (1.0f / BK) + 1.0f) + 0.5f * n * (n + 1.0f) * (float)T * (1.0f / BK)
                      : n * (float)p.most_tiles(a, T);
        }
        total += wave_sum(t);
    }
    // (one item a CU, or two where those are long)
    float c = total * 1.0001f / (float)a.budget + 1.0f;
    if (c >= LONG_TILES) c = total * 1.0001f / (2.f * (float)a.budget) + 1.0f;
    return c < (float)a.min_tiles ? a.min_tiles : c < (float)MAX_TILES ? (int)c : MAX_TILES;
}

// What a workgroup of the packed kernel does: a block's rows, over its keys.
__device__ __forceinline__ void set_block(const g3k_paged_args &a, int b, const Prompt &p, int rb, int T, Unit &u) {
    const int tok = rb * T, left = min(p.n - tok, T);
    u.b = b;
    u.run = p.first + tok;
    u.pos = p.pos + tok;
    u.count = left * a.group;
    u.kend = max(u.pos + left, 0);
    u.kbeg = max(u.pos + 1 - a.window, 0);
}
__device__ __forceinline__ int block_chunks(const Unit &u, int c) {
    const int n = u.kend > u.kbeg ? (u.kend + BK - 1) / BK - u.kbeg / BK : 0;
    return n > 0 ? (n + c - 1) / c : 1;
}
__device__ __forceinline__ Prompt uniform(const Prompt &p, int lane) {
    Prompt r;
    r.first = __builtin_amdgcn_readlane(p.first, lane);
    r.n = __builtin_amdgcn_readlane(p.n, lane);
    r.pos = __builtin_amdgcn_readlane(p.pos, lane);
    r.blocks = __builtin_amdgcn_readlane(p.blocks, lane);
    r.all = __builtin_amdgcn_readlane((int)p.all, lane) != 0;
    return r;
}

// Items of a batch of up to 64 sequences run longest first, in classes:
// whole chunks, then the last ones of blocks from 3/4, 1/2, 1/4, 1/8 of one and
// from nothing, so that the CUs end together (5 bf16 chunks behind cached
// keys 282 us, sequence by sequence 307).  Class 0 holds chunk p of blocks with
// p + 1 whole ones, class k chunk p of blocks with p c + [lo, hi) tiles.
constexpr int CLASSES = 6;
struct Classes {
    int c, T;
    // least tiles, beyond p chunks, of classes i and before
    __device__ __forceinline__ int least(int i, int p) const { return i == 0 ? c : i < 5 ? max(c * (0x1246 >> 4 * (i - 1) & 15) >> 3, 1) : p == 0 ? 0 : 1; }
    // class k's blocks of which chunk p is one: [from, to)
    __device__ __forceinline__ void blocks(const Prompt &s, int k, int p, int &from, int &to) const {
        from = s.first_of(p * c + least(k, p), T);
        to = k ? s.first_of(p * c + least(k - 1, p), T) : s.blocks;
    }
    __device__ __forceinline__ void count(const g3k_paged_args &a, const Prompt &s, int (&n)[CLASSES]) const {
#pragma unroll
        for (int k = 0; k < CLASSES; k++) n[k] = 0;
        if (s.blocks == 0) return;
        if (!s.all) {
            n[0] = s.blocks * s.chunks(a, c, T);
            return;
        }
        const int most = s.most_tiles(a, T);
        for (int p = 0; p * c <= most; p++) {
            int to = s.blocks;
#pragma unroll
            for (int k = 0; k < CLASSES; k++) {
                const int from = s.first_of(p * c + least(k, p), T);
                n[k] += to - from;
                to = from;
            }
        }
    }
};

// What workgroup `item` of the batch does: a block's rows and a chunk of its
// keys, and where the chunk's part goes: slots count chunk by chunk of each
// sequence, its last block first.  False past the last item.
__device__ bool find_item(const g3k_paged_args &a, int item, int c, int T, int lane, Unit &u, int &chunk, int &slot) {
    if (a.budget > 0 && a.s.num_seqs <= 64) {
        const Prompt mine = prompt_of(a, lane, T);
        const int slots = mine.blocks > 0 ? mine.items(a, c, T) : 0;
        const Classes classes = {c, T};
        int counts[CLASSES], before = 0;
        classes.count(a, mine, counts);
#pragma unroll
        for (int cls = 0; cls < CLASSES; cls++) {
            const int n = counts[cls], upto = wave_scan_int(n);
            const uint64_t past = __builtin_amdgcn_ballot_w64(item - before < upto);
            if (!past) {
                before += __builtin_amdgcn_readlane(upto, 63);
                continue;
            }
            const int at = __builtin_ctzll(past);
            const Prompt p = uniform(mine, at);
            int k = item - before - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(n, at)), rb;
            if (p.all) {
                for (chunk = 0;; chunk++) {
                    int from, to;
                    classes.blocks(p, cls, chunk, from, to);
                    if (k < to - from) {
                        rb = to - 1 - k;
                        break;
                    }
                    k -= to - from;
                }
            } else {
                chunk = k / p.blocks;
                rb = p.blocks - 1 - k % p.blocks;
            }
            slot = __builtin_amdgcn_readlane(wave_scan_int(slots), at) - __builtin_amdgcn_readlane(slots, at) + p.blocks - 1 - rb;
            for (int q = 0; q < chunk; q++) slot += p.blocks - p.first_with(q, c, T);
            set_block(a, at, p, rb, T, u);
            return slot < a.items;      // (not so where rows of sequences overlap)
        }
        return false;
    }
    slot = item;
    int before = 0;
    for (int base = 0; base < a.s.num_seqs; base += 64) {
        const Prompt mine = prompt_of(a, base + lane, T);
        const int n = mine.blocks > 0 ? mine.items(a, c, T) : 0;
        const int upto = wave_scan_int(n);
        const uint64_t past = __builtin_amdgcn_ballot_w64(item - before < upto);
        if (past) {
            const int at = __builtin_ctzll(past);
            const Prompt p = uniform(mine, at);
            int k = item - before - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(n, at));
            for (chunk = 0;; chunk++) {
                const int here = p.blocks - p.first_with(chunk, c, T);
                if (k < here) break;
                k -= here;
            }
            set_block(a, base + at, p, p.blocks - 1 - k, T, u);
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

template <bool BF16, int NW>
__global__ __launch_bounds__(64 * NW, NW / 4) void paged_prefill_kernel(g3k_paged_args a) {
    __shared__ __align__(16) char lds[Lds<BF16>::BYTES];
    __shared__ f32x2 factors[3 * NOTES + 64];
    __shared__ int exps[3 * NOTES + 64];
    int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = blockIdx.x % a.n_kv_heads, item = blockIdx.x / a.n_kv_heads;
    constexpr int ROWS = 16 * NW;
    Unit u;
    int chunk, part;
    const int T = ROWS / a.group, c = __builtin_amdgcn_readfirstlane(prompt_chunk(a, T, lane));
    if (!find_item(a, item, c, T, lane, u, chunk, part)) return;
    const int parts = block_chunks(u, c);
    if (chunk >= parts) return;
    const int kbeg = max(u.kbeg, (u.kbeg / BK + chunk * c) * BK), kend = min((long long)u.kend, (u.kbeg / BK + (chunk + 1LL) * c) * BK);
    Rows s;
    const int gs = __builtin_ctz(a.group);
    {
        const int row = wave * 16 + (lane & 15);
        const bool live = row < u.count;
        const int tok = row >> gs, h = head * a.group + (row & (a.group - 1));
        const int hi = u.pos + tok + 1;
        s.hi = live ? min(hi, kend) : INT_MAX;
        s.lo = live ? max(hi - a.window, kbeg) : 0;
        begin_rows(s);
        u.kbeg = kbeg;
        u.kend = kend;
        walk<BF16, NW>(a, head, u, lds, factors, exps, wave, lane,
                       a.q + ((long long)(u.run + tok) * a.n_kv_heads * a.group + h) * D, live, s);
    }
    G3K_RECOMPUTE(lane);      // no output address is kept through the walk
    {
        const int row = wave * 16 + (lane & 15);
        float *out = nullptr, *ml = nullptr;
        if (row < u.count) {
            if (parts > 1) {
                const long long slot = ((long long)part * a.n_kv_heads + head) * ROWS + row;
                out = a.part_o + slot * D;
                ml = a.part_ml + slot * 2;
            } else {
                out = a.out + ((long long)(u.run + (row >> gs)) * a.n_kv_heads * a.group + head * a.group +
                               (row & (a.group - 1))) * D;
            }
        }
        store_row(s, out, ml, lane);
    }
}

// A row's parts joined; every lane 4 dims.
struct Joined {
    f32x4 o;
    float m, l;
    __device__ __forceinline__ void clear() {
        o = (f32x4){0.f, 0.f, 0.f, 0.f};
        m = M_NONE;
        l = 0.f;
    }
    // Adds n <= 64 parts (n > 0): lane i's slot is part i's row.  The
    // statistics are one load a lane; the first outputs are on their way with
    // them.
    __device__ __forceinline__ void add(const g3k_paged_args &a, long long slot, int n, int lane) {
        constexpr int AT = 8;
        f32x4 x[AT];
        const auto fetch = [&](int i0) {
#pragma unroll
            for (int i = 0; i < AT; i++) {
                const int j = min(i0 + i, n - 1);
                const long long sj = (long long)(unsigned)__builtin_amdgcn_readlane((int)slot, j) |
                                     (long long)__builtin_amdgcn_readlane((int)(slot >> 32), j) << 32;
                x[i] = *reinterpret_cast<const f32x4 *>(a.part_o + sj * D + 4 * lane);
            }
        };
        float pm = M_NONE, pl = 0.f;
        if (lane < n) {
            const f32x2 st = *reinterpret_cast<const f32x2 *>(a.part_ml + 2 * slot);
            pm = st.x;
            pl = st.y;
        }
        fetch(0);
        const float most = top(wave_top(pm), m);
        const float w = pl * fast_exp2(pm - most), keep = fast_exp2(m - most);
        o *= keep;
        l = l * keep + wave_sum(w);
        m = most;
        for (int i0 = 0;;) {
#pragma unroll
            for (int i = 0; i < AT; i++)
                if (i0 + i < n) o += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), min(i0 + i, 63))) * x[i];
            i0 += AT;
            if (i0 >= n) break;
            fetch(i0);
        }
    }
    __device__ __forceinline__ void store(float *out, int lane) const {
        const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
        *reinterpret_cast<f32x4 *>(out + 4 * lane) = o * inv;
    }
};

// MERGE_ROWS rows of a block and head per workgroup, one wave a row.  Blocks
// of one chunk were stored whole.
constexpr int MERGE_ROWS = 8;
template <int NW>
__global__ __launch_bounds__(256) void paged_prefill_merge_kernel(g3k_paged_args a) {
    constexpr int ROWS = 16 * NW;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row0 = blockIdx.x % (ROWS / MERGE_ROWS) * MERGE_ROWS, x = blockIdx.x / (ROWS / MERGE_ROWS);
    const int head = x % a.n_kv_heads, blk = x / a.n_kv_heads;
    const int T = ROWS / a.group, c = __builtin_amdgcn_readfirstlane(prompt_chunk(a, T, lane));
    int blocks = 0, items = 0;     // before this run of sequences
    for (int base = 0; base < a.s.num_seqs; base += 64) {
        const Prompt mine = prompt_of(a, base + lane, T);
        const int n = mine.blocks > 0 ? mine.items(a, c, T) : 0;
        const int upto = wave_scan_int(mine.blocks), iupto = wave_scan_int(n);
        const uint64_t past = __builtin_amdgcn_ballot_w64(blk - blocks < upto);
        if (!past) {
            blocks += __builtin_amdgcn_readlane(upto, 63);
            items += __builtin_amdgcn_readlane(iupto, 63);
            continue;
        }
        const int at = __builtin_ctzll(past);
        const Prompt p = uniform(mine, at);
        const int rb = blk - blocks - (__builtin_amdgcn_readlane(upto, at) - p.blocks);
        const int item0 = items + __builtin_amdgcn_readlane(iupto, at) - __builtin_amdgcn_readlane(n, at) + p.blocks - 1 - rb;
        Unit u;
        set_block(a, base + at, p, rb, T, u);
        const int parts = block_chunks(u, c);
        if (parts == 1) return;
        const int gs = __builtin_ctz(a.group);
        for (int row = row0 + wave; row < min(u.count, row0 + MERGE_ROWS); row += 4) {
            Joined j;
            j.clear();
            int item = item0;
            for (int q = 0; q < parts; q += 64) {
                long long slot = 0;
                const int k = min(parts - q, 64);
                for (int i = 0; i < k; i++) {
                    if (lane == i) slot = ((long long)min(item, a.items - 1) * a.n_kv_heads + head) * ROWS + row;
                    item += p.blocks - p.first_with(q + i, c, T);
                }
                j.add(a, slot, k, lane);
            }
            j.store(a.out + ((long long)(u.run + (row >> gs)) * a.n_kv_heads * a.group + head * a.group + (row & (a.group - 1))) * D, lane);
        }
        return;
    }
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

// The work of a decode: per group and ROWS of its members' rows, the prefix's
// keys; per sequence, the keys beyond.  A wave's lanes look at 64 groups or
// sequences at a time; the first 64 of each stay in registers.
struct GroupLane {
    int first, end, p, blocks, tiles;
};
struct SeqLane {
    int kbeg, len, tiles, shares;
    int alone;       // short enough for one wave (tiles is 0 then)
};

__device__ __forceinline__ GroupLane group_lane(const g3k_paged_args &a, int i, int rows) {
    GroupLane g = {0, 0, 0, 0, 0};
    if (i < a.n_groups) {
        g.p = group_prefix(a, i, g.first, g.end);
        if (g.p > 0) {
            g.blocks = ((g.end - g.first) * a.group + rows - 1) / rows;
            g.tiles = tiles_of(prefix_begin(a, g.p), g.p);
        }
    }
    return g;
}
// Where there are more sequences than CUs, one with at most this many tiles is
// one wave's work, and a workgroup takes as many of them as it has waves.
constexpr int ALONE_TILES = 4;
__device__ __forceinline__ SeqLane seq_lane(const g3k_paged_args &a, int b) {
    SeqLane s = {0, 0, 0, 0, 0};
    if (b < a.s.num_seqs) {
        int first;
        s.len = seq_len(a.s, b);
        s.shares = seq_prefix(a, b, first);
        s.kbeg = tail_begin(a, s.len, s.shares);
        s.tiles = tiles_of(s.kbeg, s.len);
        if (a.pack && s.tiles > 0 && s.tiles <= ALONE_TILES) {
            s.alone = s.tiles;
            s.tiles = 0;
        }
    }
    return s;
}

// The units' keys are cut into chunks of about equal work, as many as make
// a.budget items per KV head (one per CU), whatever the lengths: every wave
// adds the lengths up for itself, then finds its item.  One item more than
// there are CUs costs a second round of workgroups (8 unrelated sequences, 313
// tiles: 36 us with 67 items a head, 21 with 64), so where the lengths are all
// in registers the chunks are lengthened until the count fits.  Where units
// are more than half the CUs, twice as many items as units (two a CU more at
// most), or the long ones would hardly be cut (48 sequences in 3 groups, bf16:
// 77 us; 1.5 times as many 79, as many 148, 2.5 times 91).
struct DecodePlan {
    GroupLane g0;
    SeqLane s0;
    int per;        // tiles a chunk, at most; a prefix's tile counts as two
    int alone;      // sequences that are one wave's work
    __device__ __forceinline__ static int chunks(int tiles, int per) { return (tiles + per - 1) / per; }
    __device__ __forceinline__ int prefix_chunks(int tiles) const { return chunks(tiles, max((per + 1) >> 1, 1)); }

    __device__ __forceinline__ void begin(const g3k_paged_args &a, int rows, int waves, int lane) {
        g0 = group_lane(a, lane, rows);
        s0 = seq_lane(a, lane);
        const bool all = a.n_groups <= 64 && a.s.num_seqs <= 64;
        float total = 2.f * (float)g0.blocks * (float)g0.tiles + (float)s0.tiles;   // rounded: 1e-4 is added below
        int units = g0.blocks;
        alone = s0.alone > 0;
        for (int base = 64; base < a.n_groups; base += 64) {
            const GroupLane g = group_lane(a, base + lane, rows);
            total += 2.f * (float)g.blocks * (float)g.tiles;
            units += g.blocks;
        }
        for (int base = 64; base < a.s.num_seqs; base += 64) {
            const SeqLane q = seq_lane(a, base + lane);
            total += (float)q.tiles;
            alone += q.alone > 0;
        }
        total = wave_sum(total);
        alone = a.pack ? wave_sum_int(alone) : 0;
        const int packs = (alone + waves - 1) / waves;
        units = a.s.num_seqs - alone + (a.n_groups ? wave_sum_int(units) : 0);
        const int u = units + packs;
        const int budget = max(a.budget, u + min(u, 2 * a.budget)) - packs;
        const int room = all ? budget : budget - units;
        const float c = total * 1.0001f / (float)max(room, 1) + 1.0f;
        per = c < (float)a.min_tiles ? a.min_tiles : c < 2.f * MAX_TILES ? (int)c : 2 * MAX_TILES;
        if (!all) return;
        for (int i = 0; i < 16; i++) {
            if (wave_sum_int(g0.blocks * prefix_chunks(g0.tiles) + chunks(s0.tiles, per)) <= budget) break;
            per += max(per >> 3, 1);
        }
    }
};

// Chunk `item`: its unit, keys and rows, whether it is a prefix's, how many
// chunks its unit has, which of them it is, and whether its sequence shares.
// Or a pack: `alone`, and each wave finds its own sequence (chunks 0: none).
struct Found {
    bool any, prefix, alone, shares;
    int chunks, index, part;      // part: its number among the prefixes' chunks, or the tails', or the packs
};
__device__ Found find_chunk(const g3k_paged_args &a, const DecodePlan &plan, int item, int rows, int wave, int waves, int lane, Unit &u) {
    Found r = {false, false, false, false, 0, 0, item};
    const auto at = [](int v, int l) { return __builtin_amdgcn_readlane(v, l); };
    // the chunk's keys: its even share of the unit's tiles
    const auto keys = [&](int kbeg, int kend, int tiles) {
        const int each = (tiles + r.chunks - 1) / r.chunks, t0 = kbeg / BK + r.index * each;
        u.kbeg = max(kbeg, t0 * BK);
        u.kend = min(kend, (t0 + each) * BK);
    };
    const int packs = (plan.alone + waves - 1) / waves;
    if (item < packs) {      // first: one wave on its own is long at it
        r.any = r.alone = true;
        const int k = item * waves + wave;
        u.b = u.run = u.pos = u.kbeg = u.kend = 0;
        u.count = a.group;
        int before = 0;
        for (int base = 0; base < a.s.num_seqs; base += 64) {
            const SeqLane s = base ? seq_lane(a, base + lane) : plan.s0;
            const int upto = wave_scan_int(s.alone > 0);
            const uint64_t past = __builtin_amdgcn_ballot_w64(k - before < upto);
            if (past) {
                const int l = __builtin_ctzll(past);
                r.chunks = 1;
                r.shares = at(s.shares, l) > 0;
                u.b = u.run = base + l;
                u.kbeg = at(s.kbeg, l);
                u.kend = at(s.len, l);
                return r;
            }
            before += at(upto, 63);
        }
        return r;
    }
    int before = packs;
    for (int base = 0; base < a.n_groups; base += 64) {
        const GroupLane g = base ? group_lane(a, base + lane, rows) : plan.g0;
        const int c = plan.prefix_chunks(g.tiles);
        const int upto = wave_scan_int(g.blocks * c);
        const uint64_t past = __builtin_amdgcn_ballot_w64(item - before < upto);
        if (past) {
            const int l = __builtin_ctzll(past);
            const int first = at(g.first, l), end = at(g.end, l), p = at(g.p, l);
            r.chunks = at(c, l);
            const int k = item - before - (at(upto, l) - at(g.blocks, l) * r.chunks);
            const int block = k / r.chunks, left = (end - first) * a.group - block * rows;
            r.any = r.prefix = true;
            r.part = item - packs;
            r.index = k % r.chunks;
            u.b = first;
            u.run = first + block * (rows / a.group);
            u.count = left < rows ? left : rows;
            u.pos = 0;
            keys(prefix_begin(a, p), p, at(g.tiles, l));
            return r;
        }
        before += at(upto, 63);
    }
    for (int base = 0; base < a.s.num_seqs; base += 64) {
        const SeqLane s = base ? seq_lane(a, base + lane) : plan.s0;
        const int c = DecodePlan::chunks(s.tiles, plan.per);
        const int upto = wave_scan_int(c);
        const uint64_t past = __builtin_amdgcn_ballot_w64(item - before < upto);
        if (past) {
            const int l = __builtin_ctzll(past);
            r.any = true;
            r.chunks = at(c, l);
            r.index = item - before - (at(upto, l) - r.chunks);
            r.shares = at(s.shares, l) > 0;
            u.b = u.run = base + l;
            u.count = a.group;
            u.pos = 0;
            keys(at(s.kbeg, l), at(s.len, l), at(s.tiles, l));
            return r;
        }
        before += at(upto, 63);
    }
    return r;
}

// A tail chunk: one sequence's keys, for the (at most four) query heads of the
// KV head.  There is nothing to share between waves, so each takes 16 keys of
// its own at a time, straight from memory to registers to the matrix units: a
// K lane holds one key's share of every dim step's operand, a V lane four dims
// (bf16: eight) of its lane group's four keys, which are operand lanes of as
// many dim blocks, and S^T's registers are P's operand.  While the scores of
// a step are taken its V is on its way, while its values are the next K: 32
// KiB in flight a wave (bf16: 16).  The waves of a workgroup take the steps of
// one chunk in turn, or each all steps of a short sequence of its own.  The
// queries' four rows lie in LDS as operand lanes, which the other 12 columns
// of the operand read too: those columns of S^T and O^T are never used.
// Bound by bytes: 8 unrelated sequences of 37 to 4000 keys (fp32, 4 KV heads,
// 97 MB) take 30 us, 24 of them this kernel's: 3 to find the work, 15 for the
// bytes, 3 to join the waves' shares; 5 the parts' merge.  As padded 128-row
// tiles they took 62.
template <bool BF16>
struct Step {
    static constexpr int ROW = D * (BF16 ? 2 : 4);
    static constexpr int N = BF16 ? 8 : 16;        // 16-byte loads a lane and matrix
    u32x4 k[N], v[N];
    // Lane (c, g)'s offsets from the step's first row; rows outside [0, rows)
    // of it are the nearest one's.
    __device__ __forceinline__ void load_k(gbytes base, int rs, int first, int end, int lane) {
        const gbytes row = base + clampi(lane & 15, first, end - 1) * rs + (lane >> 4) * 16;
#pragma unroll
        for (int i = 0; i < N; i++) k[i] = load_global<u32x4>(row + i * 64);
    }
    __device__ __forceinline__ void load_v(gbytes base, int rs, int first, int end, int lane) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const gbytes row = base + clampi(4 * (lane >> 4) + i, first, end - 1) * rs + (lane & 15) * 16;
#pragma unroll
            for (int T = 0; T < N / 4; T++) v[T * 4 + i] = load_global<u32x4>(row + T * 256);
        }
    }
};

__device__ __forceinline__ float bf16_of(const u32x4 &x, int i) {
    const unsigned u = x[i >> 1];
    return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
}
__device__ __forceinline__ float f32_of(const u32x4 &x, int i) { return __uint_as_float(x[i]); }

template <bool BF16>
__device__ __forceinline__ int step_max(const u32x4 (&x)[BF16 ? 8 : 16]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < (BF16 ? 8 : 16); i++)
#pragma unroll
        for (int e = 0; e < (BF16 ? 8 : 4); e += 2)
            m = BF16 ? top(top(m, fabsf(bf16_of(x[i], e))), fabsf(bf16_of(x[i], e + 1)))
                     : top(top(m, fabsf(f32_of(x[i], e))), fabsf(f32_of(x[i], e + 1)));
    return wave_top_bits(m);
}

// The dim of element i of dim step kk's operand lane of group g: K's loads are
// 64 bytes of a row a group of lanes.
template <bool BF16>
__device__ __forceinline__ int step_dim(int kk, int g, int i) {
    return BF16 ? 32 * kk + 8 * g + i : 32 * kk + 16 * (i >> 2) + 4 * g + (i & 3);
}

// O^T of one row, as the waves of a workgroup leave it.
struct Tail {
    f32x4 o[16];
    float m, l;
    int ev;
};

// This wave takes steps step0, step0 + stride, ...; queries: 4 KiB, of which it
// stores the dim steps kk with kk % stride == step0.
template <bool BF16>
__device__ __forceinline__ void walk_tail(const g3k_paged_args &a, int head, const Unit &u, char *queries, int step0, int stride,
                                          int lane, Tail &s) {
    constexpr int ROW = Step<BF16>::ROW;
    const int g = lane >> 4, c = lane & 15;
    s.m = M_NONE;
    s.l = 0.f;
    s.ev = E_NONE;
#pragma unroll
    for (int d = 0; d < 16; d++) s.o[d] = (f32x4){0.f, 0.f, 0.f, 0.f};

    const int j0 = u.kbeg & ~15, steps = (u.kend - j0 + 15) / 16;
    const int *table = a.s.page_table + (long long)u.b * a.s.table_stride;
    const int shift = a.s.page_shift, mask = (1 << shift) - 1, last = max(u.kend - 1, 0) >> shift;
    const long long head_off = ((long long)head << shift) * D;
    const gbytes kb = global_bytes(a.k) + head_off * (ROW / D), vb = global_bytes(a.v) + head_off * (ROW / D);
    // lane i: the page of this wave's step base + i
    const auto look = [&](int base) { return table[min((j0 + 16 * (step0 + stride * (base + lane))) >> shift, last)]; };
    int ids = look(0);
    // the queries, row c of the group's heads: asked for before K and V, which
    // would otherwise have to arrive first
    const float *q = a.q + (((long long)u.run * a.n_kv_heads + head) * a.group + c) * D;
    const bool live = c < a.group;
    f32x4 xq[8][2];
#pragma unroll
    for (int kk = 0; kk < 8; kk++)
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const f32x4 z = {0.f, 0.f, 0.f, 0.f};
            xq[kk][i >> 2] = live ? *reinterpret_cast<const f32x4 *>(q + step_dim<BF16>(kk, g, i)) : z;
        }
    // a step's first row from the head's first page, or rows of zeros
    struct Where {
        long long off;
        int rs;
    };
    const auto where = [&](int n) {
        if ((n & 63) == 0 && n) ids = look(n);
        const unsigned page = __builtin_amdgcn_readlane(ids, n & 63);
        const int j = j0 + 16 * (step0 + stride * n);
        Where w;
        w.off = (long long)(((unsigned long long)page * (unsigned)a.page_stride + (unsigned)((j & mask) * D)) * (ROW / D));
        w.rs = page < (unsigned)a.num_pages ? ROW : 0;
        return w;
    };
    Step<BF16> x;
    const int mine = steps > step0 ? (steps - step0 + stride - 1) / stride : 0;
    const auto begin = [&](int n) { return max(u.kbeg - (j0 + 16 * (step0 + stride * n)), 0); };
    const auto end = [&](int n) { return min(u.kend - (j0 + 16 * (step0 + stride * n)), 16); };
    const gbytes zeros = global_bytes(zero_row);
    Where w = {0, 0};
    if (mine > 0) {
        w = where(0);
        x.load_k(w.rs ? kb + w.off : zeros, w.rs, begin(0), end(0), lane);
        x.load_v(w.rs ? vb + w.off : zeros, w.rs, begin(0), end(0), lane);
    }
    float qfac;
    {
        float m = 0.f;
#pragma unroll
        for (int kk = 0; kk < 8; kk++)
#pragma unroll
            for (int i = 0; i < 8; i++) m = top(m, fabsf(xq[kk][i >> 2][i & 3]));
        const int e = block_exponent(__float_as_int(col4_top(m)));
        const float sc = __builtin_amdgcn_ldexpf(1.0f, X_EXP - e);
        qfac = __builtin_amdgcn_ldexpf(a.qscale, e - X_EXP);
#pragma unroll
        for (int kk = 0; kk < 8; kk++) {
            if (kk % stride != step0 || c >= 4) continue;
            half8 h, l;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                half2v hh, ll;
                split2(xq[kk][i >> 2][i & 3], xq[kk][i >> 2][(i & 3) + 1], sc, hh, ll);
                h[i] = hh.x;
                h[i + 1] = hh.y;
                l[i] = ll.x;
                l[i + 1] = ll.y;
            }
            *reinterpret_cast<half8 *>(queries + kk * 512 + (4 * g + c) * 16) = h;
            *reinterpret_cast<half8 *>(queries + kk * 512 + 256 + (4 * g + c) * 16) = l;
        }
    }
    G3K_WAIT_BARRIER(63);
    for (int n = 0; n < mine; n++) {
        const int first = begin(n), fin = end(n);
        const bool gone = w.rs == 0;
        G3K_RECOMPUTE(lane);
        const int mk = step_max<BF16>(x.k);
        const int ek = block_exponent(mk);
        const float sk = __builtin_amdgcn_ldexpf(1.0f, X_EXP - ek);
        f32x4 sc = {0.f, 0.f, 0.f, 0.f}, sx = sc, sy = sc;
        const char *qp = queries + (4 * (lane >> 4) + (lane & 3)) * 16;
#pragma unroll
        for (int kk = 0; kk < 8; kk++) {
            const half8 qh = *reinterpret_cast<const half8 *>(qp + kk * 512);
            const half8 ql = *reinterpret_cast<const half8 *>(qp + kk * 512 + 256);
            half8 h, l;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                half2v hh, ll;
                if constexpr (BF16) {
                    hh = cvt2(bf16_of(x.k[kk], i) * sk, bf16_of(x.k[kk], i + 1) * sk);
                } else {
                    split2(f32_of(x.k[2 * kk + (i >> 2)], i & 3), f32_of(x.k[2 * kk + (i >> 2)], (i & 3) + 1), sk, hh, ll);
                    l[i] = ll.x;
                    l[i + 1] = ll.y;
                }
                h[i] = hh.x;
                h[i + 1] = hh.y;
            }
            sc = mfma(h, qh, sc);
            sx = mfma(h, ql, sx);
            if constexpr (!BF16) sy = mfma(l, qh, sy);
            KEEP_OPERANDS();
        }
        if (n + 1 < mine) {
            w = where(n + 1);
            x.load_k(w.rs ? kb + w.off : zeros, w.rs, begin(n + 1), end(n + 1), lane);
        }
        sc += sx;
        if constexpr (!BF16) sc += sy;
        const float f = qfac * __builtin_amdgcn_ldexpf(1.0f, ek - X_EXP);
        float t = M_NONE;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int j = 4 * g + r;
            sc[r] = gone || j < first || j >= fin ? -INFINITY : sc[r] * f;
            t = top(t, sc[r]);
        }
        t = col4_top(t);
        const int mv = step_max<BF16>(x.v);
        if (max(mk, mv) >= NOT_FINITE) s.l = NAN;     // every head sees the step's rows
        const int ev = block_exponent(mv);
        const bool up = t > s.m + LAZY;
        if (__builtin_amdgcn_ballot_w64(up) || ev > s.ev) {
            const float m = up ? t : s.m;
            float keep = fast_exp2(s.m - m);
            s.m = m;
            s.l *= keep;
            if (ev > s.ev) {
                keep *= s.ev == E_NONE ? 0.f : __builtin_amdgcn_ldexpf(1.0f, s.ev - ev - 2);
                s.ev = ev + 2;
            }
#pragma unroll
            for (int d = 0; d < 16; d++) s.o[d] *= keep;
        }
        const float pf = __builtin_amdgcn_ldexpf(1.0f, P_EXP + ev - s.ev), sv = __builtin_amdgcn_ldexpf(1.0f, X_EXP - ev);
        half4v ph, pl;
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
            const float p0 = fast_exp2(sc[r] - s.m), p1 = fast_exp2(sc[r + 1] - s.m);
            s.l += p0 + p1;
            half2v h, l;
            split2(p0, p1, pf, h, l);
            ph[r] = h.x;
            ph[r + 1] = h.y;
            pl[r] = l.x;
            pl[r + 1] = l.y;
        }
        constexpr int PER = BF16 ? 8 : 4;       // dims a lane and load
        half4v lo = {};
#pragma unroll
        for (int d = 0; d < 16; d++) {
            const int T = d / PER, e = d % PER;
            half4v h, l;
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                half2v hh, ll;
                if constexpr (BF16) {
                    hh = cvt2(bf16_of(x.v[T * 4 + i], e) * sv, bf16_of(x.v[T * 4 + i + 1], e) * sv);
                } else {
                    split2(f32_of(x.v[T * 4 + i], e), f32_of(x.v[T * 4 + i + 1], e), sv, hh, ll);
                    l[i] = ll.x;
                    l[i + 1] = ll.y;
                }
                h[i] = hh.x;
                h[i + 1] = hh.y;
            }
            s.o[d] = __builtin_amdgcn_mfma_f32_16x16x16f16(h, ph, s.o[d], 0, 0, 0);
            if constexpr (!BF16) {
                if (d > 0) s.o[d - 1] = __builtin_amdgcn_mfma_f32_16x16x16f16(lo, ph, s.o[d - 1], 0, 0, 0);
                lo = l;
            }
            s.o[d] = __builtin_amdgcn_mfma_f32_16x16x16f16(h, pl, s.o[d], 0, 0, 0);
        }
        if constexpr (!BF16) s.o[15] = __builtin_amdgcn_mfma_f32_16x16x16f16(lo, ph, s.o[15], 0, 0, 0);
        if (n + 1 < mine) x.load_v(w.rs ? vb + w.off : zeros, w.rs, begin(n + 1), end(n + 1), lane);
    }
}

// Stores a tail's row of this lane (c < group): rows stride D apart, normalised.
template <bool BF16>
__device__ __forceinline__ void store_tail_rows(const Tail &s, float inv, float *rows, int lane) {
    const int c = lane & 15, g = lane >> 4;
    const int e = s.ev == E_NONE ? 0 : s.ev - X_EXP - P_EXP;
    constexpr int PER = BF16 ? 8 : 4;
#pragma unroll
    for (int T = 0; T < 16 / PER; T++)
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int t = 0; t < PER; t += 4) {
                f32x4 x;
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = __builtin_amdgcn_ldexpf(s.o[PER * T + t + i][r] * inv, e);
                *reinterpret_cast<f32x4 *>(rows + c * D + 16 * PER * T + PER * (4 * g + r) + t) = x;
            }
}

// Joins the waves' shares of a tail and stores the group's rows: to out, or a
// part with its (max, sum).
template <bool BF16, int NW>
__device__ __forceinline__ void store_tail(const g3k_paged_args &a, Tail &s, char *lds, int wave, int lane, float *out, float *ml) {
    float *ws = reinterpret_cast<float *>(lds);            // [wave][row][D], then [wave][row] of (max, sum)
    float *st = ws + NW * 4 * D;
    const int c = lane & 15, g = lane >> 4;
    const float l = col4_sum(s.l);
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
    __syncthreads();           // the queries in LDS have been read
    if (c < a.group) {
        store_tail_rows<BF16>(s, inv, ws + wave * 4 * D, lane);
        if (g == 0) {
            st[2 * (wave * 4 + c)] = s.m;
            st[2 * (wave * 4 + c) + 1] = l;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.group * (D / 4); i += 64 * NW) {
        const int row = i / (D / 4), d = i % (D / 4) * 4;
        float most = M_NONE;
#pragma unroll
        for (int w = 0; w < NW; w++) most = top(most, st[2 * (w * 4 + row)]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float k = st[2 * (w * 4 + row) + 1] * fast_exp2(st[2 * (w * 4 + row)] - most);
            sum += k;
            o += k * *reinterpret_cast<const f32x4 *>(ws + (w * 4 + row) * D + d);
        }
        const float y = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
        *reinterpret_cast<f32x4 *>(out + row * D + d) = o * y;
        if (ml && d == 0) {
            ml[2 * row] = most;
            ml[2 * row + 1] = sum;
        }
    }
}

constexpr int DECODE_WAVES = G3K_PAGED_DECODE_ROWS / 16;
template <bool BF16>
__global__ __launch_bounds__(64 * DECODE_WAVES, DECODE_WAVES / 4) void paged_decode_kernel(g3k_paged_args a) {
    constexpr int NW = DECODE_WAVES;
    __shared__ __align__(16) char lds[Lds<BF16>::BYTES];
    __shared__ f32x2 factors[3 * NOTES + 64];
    __shared__ int exps[3 * NOTES + 64];
    constexpr int ROWS = 16 * NW;
    int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int head = blockIdx.x % a.n_kv_heads, item = blockIdx.x / a.n_kv_heads;
    DecodePlan plan;
    plan.begin(a, ROWS, NW, lane);
    Unit u;
    const Found f = find_chunk(a, plan, item, ROWS, wave, NW, lane, u);
    if (!f.any) return;
    // Parts lie by what they are of, prefixes' chunks, tails' and packs: rows
    // a part and head.  The directory has a first part's first row, the
    // chunks, the sequence that has that row, and the rows a part.
    const int per = f.prefix ? ROWS : f.alone ? NW * a.group : a.group;
    if (f.prefix && f.part >= a.prefix_parts) return;      // (not so unless groups overlap)
    const long long first0 = (f.prefix ? 0ll : (long long)a.prefix_parts * ROWS + (f.alone ? (long long)a.items * a.group : 0ll)) * a.n_kv_heads +
                             (long long)f.part * a.n_kv_heads * per;
    const long long slot0 = first0 + head * per;
    int *dir = (f.prefix ? a.dir_prefix : a.dir_tail) + 4 * u.run;
    if (f.alone) {
        Tail s;
        walk_tail<BF16>(a, head, u, lds + wave * 4096, 0, 1, lane, s);
        if (f.chunks == 0) return;
        const float l = col4_sum(s.l);
        float *out = f.shares ? a.part_o + (slot0 + wave * a.group) * D : a.out + ((long long)u.run * a.n_kv_heads + head) * a.group * D;
        if ((lane & 15) < a.group) {
            store_tail_rows<BF16>(s, l > 0.f || l != l ? 1.0f / l : 0.f, out, lane);
            if (f.shares && lane < 16) *reinterpret_cast<f32x2 *>(a.part_ml + 2 * (slot0 + wave * a.group + lane)) = (f32x2){s.m, l};
        }
        if (head == 0 && lane == 0)
            *reinterpret_cast<u32x4 *>(dir) = (u32x4){(unsigned)first0 + wave * a.group, 1, (unsigned)u.run, (unsigned)per};
        return;
    }
    if (f.index == 0 && head == 0 && (int)threadIdx.x < (f.prefix ? u.count / a.group : 1))
        *reinterpret_cast<u32x4 *>(dir + 4 * threadIdx.x) =
            (u32x4){(unsigned)first0, (unsigned)f.chunks, (unsigned)u.run, (unsigned)per};
    if (!f.prefix) {
        Tail s;
        walk_tail<BF16>(a, head, u, lds, wave, NW, lane, s);
        // (an even share may leave the last chunk without keys: its part is empty)
        const bool whole = f.chunks == 1 && !f.shares;
        store_tail<BF16, NW>(a, s, lds, wave, lane,
                             whole ? a.out + ((long long)u.run * a.n_kv_heads + head) * a.group * D : a.part_o + slot0 * D,
                             whole ? nullptr : a.part_ml + slot0 * 2);
        return;
    }
    Rows s;
    const int gs = __builtin_ctz(a.group);
    {
        const int row = wave * 16 + (lane & 15);
        const bool live = row < u.count;
        const int seq = u.run + (row >> gs), h = head * a.group + (row & (a.group - 1));
        const int len = live ? seq_len(a.s, seq) : 0;
        s.hi = live ? min(len, u.kend) : INT_MAX;
        s.lo = live ? max(len - a.window, u.kbeg) : 0;
        begin_rows(s);
        walk<BF16, NW>(a, head, u, lds, factors, exps, wave, lane, a.q + ((long long)seq * a.n_kv_heads * a.group + h) * D, live, s);
    }
    G3K_RECOMPUTE(lane);      // no output address is kept through the walk
    const int row = wave * 16 + (lane & 15);
    const long long slot = slot0 + row;
    store_row(s, row < u.count ? a.part_o + slot * D : nullptr, a.part_ml + slot * 2, lane);
}

// One wave per sequence and query head.
__global__ __launch_bounds__(256) void paged_decode_merge_kernel(g3k_paged_args a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int heads = a.n_kv_heads * a.group;
    const long long id = (long long)blockIdx.x * 4 + wave;
    if (id >= (long long)a.s.num_seqs * heads) return;
    const int b = (int)(id / heads), h = (int)(id % heads);
    const int kvh = h / a.group, hg = h % a.group;
    // (the directories are kept within the parts whatever they hold: a batch
    // whose group bounds overlap leaves entries unwritten)
    const u32x4 dt = *reinterpret_cast<const u32x4 *>(a.dir_tail + 4 * b);
    u32x4 dp = {0, 0, 0, 0};
    if (a.n_groups > 0) dp = *reinterpret_cast<const u32x4 *>(a.dir_prefix + 4 * b);
    int first;
    const int len = seq_len(a.s, b), p = seq_prefix(a, b, first);
    const bool tail = tiles_of(tail_begin(a, len, p), len) > 0;
    if (p == 0 && tail && dt.y == 1) return;        // written by its one chunk
    Joined j;
    j.clear();
    const auto add = [&](u32x4 d) {
        const long long slot = (long long)d.x + (long long)kvh * d.w + (long long)(b - (int)d.z) * a.group + hg;
        const long long stride = (long long)a.n_kv_heads * d.w;
        const int n = clampi((int)d.y, 1, a.items);
        for (int q = 0; q < n; q += 64) {
            const long long at = slot + (q + min(lane, n - 1 - q)) * stride;
            j.add(a, at < 0 || at >= a.part_rows ? 0 : at, min(n - q, 64), lane);
        }
    };
    if (tail) add(dt);
    if (p > 0) add(dp);
    j.store(a.out + id * D, lane);
}

}  // namespace

namespace {

template <bool BF16, int NW>
void launch_prefill(const g3k_paged_args &a, unsigned wgs, hipStream_t st) {
    hipLaunchKernelGGL((paged_prefill_kernel<BF16, NW>), dim3(wgs), dim3(64 * NW), 0, st, a);
    const unsigned merges = (unsigned)a.blocks * a.n_kv_heads * (16 * NW / MERGE_ROWS);
    if (a.budget > 0) hipLaunchKernelGGL(paged_prefill_merge_kernel<NW>, dim3(merges), dim3(256), 0, st, a);
}

template <bool BF16>
void launch_decode(const g3k_paged_args &a, unsigned wgs, hipStream_t st) {
    hipLaunchKernelGGL(paged_decode_kernel<BF16>, dim3(wgs), dim3(64 * DECODE_WAVES), 0, st, a);
    const unsigned merges = ((unsigned)a.s.num_seqs * a.n_kv_heads * a.group + 3) / 4;
    hipLaunchKernelGGL(paged_decode_merge_kernel, dim3(merges), dim3(256), 0, st, a);
}

}  // namespace

extern "C" int g3k_paged_prefill(const g3k_paged_args *a, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    const long long wgs = (long long)a->items * a->n_kv_heads;
    if (wgs * 16 > INT_MAX) return (int)hipErrorInvalidValue;
    const unsigned n = (unsigned)wgs;
    if (a->waves == 8) a->bf16 ? launch_prefill<true, 8>(*a, n, st) : launch_prefill<false, 8>(*a, n, st);
    else a->bf16 ? launch_prefill<true, 4>(*a, n, st) : launch_prefill<false, 4>(*a, n, st);
    return (int)hipGetLastError();
}

extern "C" int g3k_paged_decode(const g3k_paged_args *a, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    const long long wgs = (long long)a->items * a->n_kv_heads;
    if (wgs > INT_MAX || (long long)a->s.num_seqs * a->n_kv_heads * a->group > INT_MAX) return (int)hipErrorInvalidValue;
    a->bf16 ? launch_decode<true>(*a, (unsigned)wgs, st) : launch_decode<false>(*a, (unsigned)wgs, st);
    return (int)hipGetLastError();
}
