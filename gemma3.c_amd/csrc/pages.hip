// pages.hip - a KV cache in pages: writing packed tokens into it, and forking
// and compacting the sequences it holds.
//
// paged_write: per head y = x / sqrt(mean x^2 + eps) (1 + w), then the
// rotation (a, b) -> (a c - b s, a s + b c) of dims (i, i + 128) by the
// table's row of the token's position: q to q_out, k and v to the row of the
// token's page (bf16 pages round to nearest even).  Bound by bytes.  Half a
// wave holds a 256-float head vector, 4 dims and their 4 partners a lane, so
// both loads and the rotation's table row are 16 bytes a lane and the
// rotation stays inside the lane; a wave takes four vectors of a token, so
// its sequence, position and table row are looked up once for four.  8192
// tokens into bf16 pages, 243 MB: 46 us, 5.3 TB/s (a large copy reaches 4.8);
// 48 single tokens 4.9 us, one launch.
//
// pages_fork: child b continues sequence parent[b], add[b] tokens longer (or
// shorter).  Pages are shared; a page that a child is going to write (the
// partial last one) has to be its own, so it is copied unless nobody else
// keeps it.  How many sequences hold a page is counted anew from the tables
// in each call, so there are no counters to keep in step: a page that no
// table names (and the caller does not hold) is free.  Free pages are handed
// out in ascending order to children in ascending order: the result does not
// depend on timing.
//
// pages_compact: the pages in use move to the lowest numbers.
//
// Both are integers over tables (latency: two to four launches), then copies of
// rows of every layer's K and V (bytes): 256 samples of 32 prompts over 34
// layers, 2.4 GB, 417 us, 5.8 TB/s; a pool of 2500 pages with 5.5 GB to move
// 1149 us, 4.8 TB/s; a beam step of 16 children 10 us.
#include <hip/hip_runtime.h>
#include <limits.h>

#include "g3k.h"
#include "g3k_device.h"
#include "paged_body.h"

namespace {

using namespace g3k;
constexpr int D = G3K_HEAD_DIM;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}

// ---- writing tokens -------------------------------------------------------------

// The sequence that packed row i belongs to: the last that begins at or
// before it, found 64 candidates at a time; -1 where no sequence has it.
__device__ int seq_of_row(const g3k_paged_seqs &s, int i, int lane) {
    if (!s.q_start) return i < s.num_seqs ? i : -1;
    int lo = 0, n = s.num_seqs;
    for (;;) {
        const int step = (n + 63) / 64;
        const int at = lane * step;
        const bool le = at < n && s.q_start[lo + at] <= i;
        const uint64_t m = __builtin_amdgcn_ballot_w64(le);
        if (!m) return -1;
        const int k = 63 - __builtin_clzll(m);
        lo += k * step;
        n = n - k * step < step ? n - k * step : step;
        if (step == 1) break;
    }
    int first, rows;
    seq_rows(s, lo, first, rows);
    return i >= first && i < first + rows ? lo : -1;
}

// Sum over a half wave's 32 lanes.
__device__ __forceinline__ float half_sum(float v) { return pair16_sum(row16_sum(v)); }

constexpr int WRITE_VECS = 4;   // head vectors per wave

template <bool BF16>
__global__ __launch_bounds__(256) void paged_write_kernel(g3k_paged_write_args a) {
    const int lane = threadIdx.x & 63, l32 = lane & 31;
    const long long wid = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int heads = a.group * a.n_kv_heads, nvec = heads + 2 * a.n_kv_heads;
    const int parts = (nvec + WRITE_VECS - 1) / WRITE_VECS;
    const long long tok = wid / parts;
    if (tok >= a.s.total_q) return;
    const int i = (int)tok, v0 = (int)(wid % parts) * WRITE_VECS;
    f32x4 x[WRITE_VECS / 2], y[WRITE_VECS / 2];
#pragma unroll
    for (int u = 0; u < WRITE_VECS / 2; u++) {
        const int v = min(v0 + 2 * u + (lane >> 5), nvec - 1);
        const float *src = v < heads                  ? a.Q + ((long long)i * heads + v) * D
                           : v < heads + a.n_kv_heads ? a.K + ((long long)i * a.n_kv_heads + v - heads) * D
                                                      : a.V + ((long long)i * a.n_kv_heads + v - heads - a.n_kv_heads) * D;
        x[u] = *reinterpret_cast<const f32x4 *>(src + 4 * l32);
        y[u] = *reinterpret_cast<const f32x4 *>(src + 128 + 4 * l32);
    }
    const int b = __builtin_amdgcn_readfirstlane(seq_of_row(a.s, i, lane));
    if (b < 0) return;
    int first, n;
    seq_rows(a.s, b, first, n);
    const int pos = __builtin_amdgcn_readfirstlane(seq_len(a.s, b) - n + (i - first));
    if (pos < 0 || pos >= a.max_context) return;
    const int page = __builtin_amdgcn_readfirstlane(a.s.page_table[(long long)b * a.s.table_stride + (pos >> a.s.page_shift)]);
    const int row = pos & ((1 << a.s.page_shift) - 1);
    const f32x4 r0 = *reinterpret_cast<const f32x4 *>(a.rope + (long long)pos * D + 8 * l32);
    const f32x4 r1 = *reinterpret_cast<const f32x4 *>(a.rope + (long long)pos * D + 8 * l32 + 4);
    const f32x4 c = {r0.x, r0.z, r1.x, r1.z}, s = {r0.y, r0.w, r1.y, r1.w};
#pragma unroll
    for (int u = 0; u < WRITE_VECS / 2; u++) {
        const int v = v0 + 2 * u + (lane >> 5);
        const int kind = v < heads ? 0 : v < heads + a.n_kv_heads ? 1 : 2;
        f32x4 p = x[u], q = y[u];
        if (a.q_norm) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) ss += p[e] * p[e] + q[e] * q[e];
            const float inv = 1.0f / sqrtf(half_sum(ss) / (float)D + a.eps);
            const uint16_t *w = kind == 1 ? a.k_norm : a.q_norm;
            const u32x2 wp = *reinterpret_cast<const u32x2 *>(w + 4 * l32), wq = *reinterpret_cast<const u32x2 *>(w + 128 + 4 * l32);
            if (kind != 2) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t a16 = wp[e >> 1] >> (16 * (e & 1)), b16 = wq[e >> 1] >> (16 * (e & 1));
                    p[e] = p[e] * inv * (1.0f + bf16f(a16 & 0xffff));
                    q[e] = q[e] * inv * (1.0f + bf16f(b16 & 0xffff));
                }
            }
        }
        if (kind != 2) {
            const f32x4 t = p * c - q * s;
            q = p * s + q * c;
            p = t;
        }
        if (v >= nvec) continue;
        if (kind == 0) {
            float *dst = a.q_out + ((long long)i * heads + v) * D;
            *reinterpret_cast<f32x4 *>(dst + 4 * l32) = p;
            *reinterpret_cast<f32x4 *>(dst + 128 + 4 * l32) = q;
        } else if ((unsigned)page < (unsigned)a.num_pages) {
            const int h = v - heads - (kind == 2 ? a.n_kv_heads : 0);
            const long long off = page * a.page_stride + (((long long)h << a.s.page_shift) + row) * D;
            void *base = kind == 1 ? a.k : a.v;
            if constexpr (BF16) {
                uint16_t *dst = static_cast<uint16_t *>(base) + off;
                *reinterpret_cast<u32x2 *>(dst + 4 * l32) = (u32x2){bf16_pair(p.x, p.y), bf16_pair(p.z, p.w)};
                *reinterpret_cast<u32x2 *>(dst + 128 + 4 * l32) = (u32x2){bf16_pair(q.x, q.y), bf16_pair(q.z, q.w)};
            } else {
                float *dst = static_cast<float *>(base) + off;
                *reinterpret_cast<f32x4 *>(dst + 4 * l32) = p;
                *reinterpret_cast<f32x4 *>(dst + 128 + 4 * l32) = q;
            }
        }
    }
}

// ---- counting -------------------------------------------------------------------

// Per page: how many sequences hold it, and of children that are going to write
// it how many there are and the first one.
struct Counts {
    int *ref, *writers, *first;
};

// Counts start from the caller's own holds.
__device__ __forceinline__ void clear_page(const g3k_pages_args &a, const Counts &n, int p) {
    n.ref[p] = a.held && a.held[p] ? 1 : 0;
    if (n.writers) {
        n.writers[p] = 0;
        n.first[p] = INT_MAX;
    }
    if (a.map) a.map[p] = p;
}
__global__ __launch_bounds__(256) void pages_clear_kernel(g3k_pages_args a) {
    const int p = blockIdx.x * 256 + threadIdx.x;
    if (p < a.num_pages) clear_page(a, {a.ref, a.writers, a.first}, p);
}

__device__ __forceinline__ int pages_of(int n, int shift) { return (n + (1 << shift) - 1) >> shift; }

// One wave: what child b keeps of its parent, and its claim on the last page if
// it is going to write there.
__device__ void count_child(const g3k_pages_args &a, const Counts &n, int b, int lane) {
    const int cap = a.table_stride << a.page_shift;
    const int p = a.parent ? a.parent[b] : b;
    const bool real = p >= 0 && p < a.n_in;
    const int old = real ? clampi(a.len_in[p], 0, cap) : 0;
    long long want = real ? (long long)old + (a.add ? a.add[b] : 0) : 0;
    if (want < 0) want = 0;
    const bool fits = want <= cap;
    if (!fits) want = old;
    const int keep = want < old ? (int)want : old;
    const int kept = pages_of(keep, a.page_shift);
    const int *row = a.table_in + (long long)(real ? p : 0) * a.table_stride;
    int *mine = a.rows + (long long)b * a.table_stride;
    for (int j = lane; j < kept; j += 64) {
        const int page = row[j];
        mine[j] = page;
        if ((unsigned)page < (unsigned)a.num_pages) atomicAdd(&n.ref[page], 1);
    }
    if (lane) return;
    int tail = -1;
    if (want > old && (old & ((1 << a.page_shift) - 1))) {
        tail = row[old >> a.page_shift];
        if ((unsigned)tail < (unsigned)a.num_pages) {
            atomicAdd(&n.writers[tail], 1);
            atomicMin(&n.first[tail], b);
        } else {
            tail = -1;      // no page to copy: the entry stays as it is
        }
    }
    g3k_fork_child c;
    c.old_len = old;
    c.want = (int)want;
    c.kept = kept;
    c.full = pages_of((int)want, a.page_shift);
    c.tail = tail;
    c.offset = 0;
    c.granted = fits;
    c.copy = 0;
    a.child[b] = c;
}
__global__ __launch_bounds__(256) void fork_count_kernel(g3k_pages_args a) {
    const int b = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (b < a.n_out) count_child(a, {a.ref, a.writers, a.first}, b, threadIdx.x & 63);
}

__device__ void count_sequence(const g3k_pages_args &a, int *ref, int b, int lane) {
    const int n = pages_of(clampi(a.len_in[b], 0, a.table_stride << a.page_shift), a.page_shift);
    const int *row = a.table_in + (long long)b * a.table_stride;
    for (int j = lane; j < n; j += 64) {
        const int page = row[j];
        if ((unsigned)page < (unsigned)a.num_pages) atomicAdd(&ref[page], 1);
    }
}
__global__ __launch_bounds__(256) void compact_count_kernel(g3k_pages_args a) {
    const int b = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (b < a.n_in) count_sequence(a, a.ref, b, threadIdx.x & 63);
}

// ---- one workgroup over all pages ---------------------------------------------------

constexpr int PLAN_T = 1024, PLAN_W = PLAN_T / 64;

// Sum of the waves' counts before this wave, and of all.
__device__ __forceinline__ int waves_before(int mine, int *slot, int wave, int lane, int &total) {
    __syncthreads();
    if (lane == 0) slot[wave] = mine;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < PLAN_W; w++) {
        if (w < wave) before += slot[w];
        total += slot[w];
    }
    return before;
}

// The pages that one wave looks at: a run of whole 64s.
__device__ __forceinline__ void wave_pages(int num_pages, int wave, int &begin, int &end) {
    const int per = (num_pages + PLAN_T - 1) / PLAN_T * 64;
    const long long b = (long long)wave * per, e = b + per;
    begin = b < num_pages ? (int)b : num_pages;
    end = e < num_pages ? (int)e : num_pages;
}

// Lists, in ascending order from list[0], the pages of [begin, end) that
// `is` names; at: how many before this wave's.  At most `most` are listed.
template <typename F>
__device__ __forceinline__ int list_pages(int begin, int end, int lane, int *list, int at, int most, F is) {
    for (int p = begin; p < end; p += 64) {
        const bool yes = p + lane < end && is(p + lane);
        const uint64_t m = __builtin_amdgcn_ballot_w64(yes);
        const int k = at + __builtin_popcountll(m & ((1ull << lane) - 1));
        if (yes && list && k < most) list[k] = p + lane;
        at += __builtin_popcountll(m);
    }
    return at;
}

// Who copies its last page, how many pages each child needs, which children
// get theirs, and the free pages in order.
__device__ void plan_fork(const g3k_pages_args &a, const Counts &n, int *slot) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int begin, end, nfree, before, total;
    wave_pages(a.num_pages, wave, begin, end);
    const int *ref = n.ref;
    const int mine = list_pages(begin, end, lane, nullptr, 0, 0, [ref](int p) { return ref[p] == 0; });
    const int free_before = waves_before(mine, slot, wave, lane, nfree);
    int needed = 0, given = 0, refused = 0;
    for (int base = 0; base < a.n_out; base += PLAN_T) {
        const int b = base + threadIdx.x;
        g3k_fork_child c = {0, 0, 0, 0, -1, 0, 1, 0};
        int need = 0;
        if (b < a.n_out) {
            c = a.child[b];
            // the first child to write a page that all who hold it are going
            // to write keeps it; the others, and everyone where somebody
            // keeps it as it is, take a copy
            c.copy = c.tail >= 0 && !(n.first[c.tail] == b && n.writers[c.tail] == n.ref[c.tail]);
            need = c.full - c.kept + c.copy;
        }
        const int upto = wave_scan_int(need);
        before = waves_before(__shfl(upto, 63), slot, wave, lane, total);
        c.offset = needed + before + upto - need;
        needed = total > INT_MAX - needed ? INT_MAX : needed + total;
        c.granted = c.granted && (need == 0 || (c.offset >= 0 && need <= nfree - c.offset));
        if (b < a.n_out) {
            if (!c.granted) {
                c.want = c.old_len;
                c.full = c.kept;
                c.copy = 0;
                need = 0;
            }
            a.child[b] = c;
            given += need;
            refused += !c.granted;
        }
    }
    list_pages(begin, end, lane, a.list, free_before, needed, [ref](int p) { return ref[p] == 0; });
    int all_given, all_refused;
    (void)waves_before(wave_sum_int(given), slot, wave, lane, all_given);
    (void)waves_before(wave_sum_int(refused), slot, wave, lane, all_refused);
    if (threadIdx.x == 0 && a.status) {
        a.status[0] = a.num_pages - nfree + all_given;
        a.status[1] = all_refused;
    }
}

// The pages in use from number `used` on, and the free ones below, in order:
// the k-th of the one moves to the k-th of the other.
__device__ void plan_compaction(const g3k_pages_args &a, const int *ref, int *slot) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int begin, end, used, moves, holes;
    wave_pages(a.num_pages, wave, begin, end);
    const int *held = a.held;
    const int mine = list_pages(begin, end, lane, nullptr, 0, 0, [ref](int p) { return ref[p] != 0; });
    (void)waves_before(mine, slot, wave, lane, used);
    const auto moved = [ref, held, used](int p) { return p >= used && ref[p] != 0 && !(held && held[p]); };
    const auto hole = [ref, used](int p) { return p < used && ref[p] == 0; };
    const int m0 = waves_before(list_pages(begin, end, lane, nullptr, 0, 0, moved), slot, wave, lane, moves);
    const int h0 = waves_before(list_pages(begin, end, lane, nullptr, 0, 0, hole), slot, wave, lane, holes);
    list_pages(begin, end, lane, a.list, m0, a.num_pages, moved);
    list_pages(begin, end, lane, a.list2, h0, a.num_pages, hole);
    __threadfence_block();
    __syncthreads();
    // there are at least as many holes as pages to move
    for (int k = threadIdx.x; k < moves; k += PLAN_T) a.map[a.list[k]] = a.list2[k];
    if (threadIdx.x == 0) {
        a.count[0] = moves;
        if (a.status) {
            a.status[0] = used;
            a.status[1] = moves;
        }
    }
}

__global__ __launch_bounds__(PLAN_T) void fork_plan_kernel(g3k_pages_args a) {
    __shared__ int slot[PLAN_W];
    plan_fork(a, {a.ref, a.writers, a.first}, slot);
}
__global__ __launch_bounds__(PLAN_T) void compact_plan_kernel(g3k_pages_args a) {
    __shared__ int slot[PLAN_W];
    plan_compaction(a, a.ref, slot);
}

// A small pool and few sequences: the counts are in LDS, and one launch takes
// the place of three.  A wave counts two sequences at most, one after the
// other (16 children, 2048 pages: 10.2 us against 14.3; 256 children in 1024
// pages counted so as well, 434 against 420).
constexpr int SMALL_PAGES = 4096, SMALL_SEQS = 2 * PLAN_W;
__global__ __launch_bounds__(PLAN_T) void fork_small_kernel(g3k_pages_args a) {
    __shared__ int slot[PLAN_W], ref[SMALL_PAGES], writers[SMALL_PAGES], first[SMALL_PAGES];
    const Counts n = {ref, writers, first};
    for (int p = threadIdx.x; p < a.num_pages; p += PLAN_T) clear_page(a, n, p);
    __syncthreads();
    for (int b = threadIdx.x >> 6; b < a.n_out; b += PLAN_W) count_child(a, n, b, threadIdx.x & 63);
    __threadfence_block();
    __syncthreads();
    plan_fork(a, n, slot);
}
__global__ __launch_bounds__(PLAN_T) void compact_small_kernel(g3k_pages_args a) {
    __shared__ int slot[PLAN_W], ref[SMALL_PAGES];
    for (int p = threadIdx.x; p < a.num_pages; p += PLAN_T) clear_page(a, {ref, nullptr, nullptr}, p);
    __syncthreads();
    for (int b = threadIdx.x >> 6; b < a.n_in; b += PLAN_W) count_sequence(a, ref, b, threadIdx.x & 63);
    __threadfence_block();
    __syncthreads();
    plan_compaction(a, ref, slot);
}

// ---- tables and copies ----------------------------------------------------------

// Copies `bytes` (a multiple of 16) with the workgroup's threads.
__device__ __forceinline__ void copy_bytes(char *dst, const char *src, long long bytes) {
    for (long long o = (long long)threadIdx.x * 16; o < bytes; o += 256 * 16)
        *reinterpret_cast<u32x4 *>(dst + o) = *reinterpret_cast<const u32x4 *>(src + o);
}

// Workgroups (b, 0): child b's table row and length.  All (b, y): the rows of
// its copied page in layer y / 2's K (y even) or V.
__global__ __launch_bounds__(256) void fork_apply_kernel(g3k_pages_args a) {
    const int b = blockIdx.x;
    const g3k_fork_child c = a.child[b];
    if (blockIdx.y == 0) {
        const int *mine = a.rows + (long long)b * a.table_stride;
        int *out = a.table_out + (long long)b * a.table_stride;
        const int own = c.copy ? c.old_len >> a.page_shift : -1;
        for (int j = threadIdx.x; j < a.table_stride; j += 256) {
            int page = -1;
            if (j == own) page = a.list[c.offset];
            else if (j < c.kept) page = mine[j];
            else if (j < c.full) page = a.list[c.offset + c.copy + j - c.kept];
            out[j] = page;
        }
        if (threadIdx.x == 0) a.len_out[b] = c.want;
    }
    if (!c.copy) return;
    const int layer = blockIdx.y >> 1;
    char *base = static_cast<char *>((blockIdx.y & 1) ? a.v : a.k) + layer * a.layer_stride * a.elem;
    const char *src = base + c.tail * a.page_stride * a.elem;
    char *dst = base + a.list[c.offset] * a.page_stride * a.elem;
    const long long head = ((long long)D << a.page_shift) * a.elem;
    const long long rows = (long long)(c.old_len & ((1 << a.page_shift) - 1)) * D * a.elem;
    for (int h = 0; h < a.n_kv_heads; h++) copy_bytes(dst + h * head, src + h * head, rows);
}

__global__ __launch_bounds__(256) void compact_apply_kernel(g3k_pages_args a) {
    if ((int)blockIdx.x < a.n_in) {
        const int b = blockIdx.x;
        const int len = clampi(a.len_in[b], 0, a.table_stride << a.page_shift);
        const int n = pages_of(len, a.page_shift);
        const long long row = (long long)b * a.table_stride;
        for (int j = threadIdx.x; j < a.table_stride; j += 256) {
            const int page = j < n ? a.table_in[row + j] : -1;
            a.table_out[row + j] = (unsigned)page < (unsigned)a.num_pages ? a.map[page] : page;
        }
        __syncthreads();      // the length may be read and written in one place
        if (threadIdx.x == 0) a.len_out[b] = len;
        return;
    }
    const long long items = (long long)a.count[0] * a.num_layers * 2;
    const long long bytes = ((long long)a.n_kv_heads * D << a.page_shift) * a.elem;
    for (long long i = blockIdx.x - a.n_in; i < items; i += gridDim.x - a.n_in) {
        const int k = (int)(i / (a.num_layers * 2)), y = (int)(i % (a.num_layers * 2));
        char *base = static_cast<char *>((y & 1) ? a.v : a.k) + (y >> 1) * a.layer_stride * a.elem;
        copy_bytes(base + a.list2[k] * a.page_stride * a.elem, base + a.list[k] * a.page_stride * a.elem, bytes);
    }
}

}  // namespace

extern "C" int g3k_paged_write(const g3k_paged_write_args *a, void *stream) {
    const int nvec = a->group * a->n_kv_heads + 2 * a->n_kv_heads;
    const long long waves = (long long)a->s.total_q * ((nvec + WRITE_VECS - 1) / WRITE_VECS);
    if (waves <= 0) return 0;
    const long long blocks = (waves + 3) / 4;
    if (blocks > UINT_MAX / 256) return (int)hipErrorInvalidValue;      // threads of a launch
    if (a->bf16)
        hipLaunchKernelGGL(paged_write_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *a);
    else
        hipLaunchKernelGGL(paged_write_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, *a);
    return (int)hipGetLastError();
}

extern "C" int g3k_pages_fork(const g3k_pages_args *a, void *stream) {
    hipStream_t s = (hipStream_t)stream;
    if (a->num_pages <= SMALL_PAGES && a->n_out <= SMALL_SEQS) {
        hipLaunchKernelGGL(fork_small_kernel, dim3(1), dim3(PLAN_T), 0, s, *a);
    } else {
        hipLaunchKernelGGL(pages_clear_kernel, dim3((a->num_pages + 255) / 256), dim3(256), 0, s, *a);
        hipLaunchKernelGGL(fork_count_kernel, dim3((a->n_out + 3) / 4), dim3(256), 0, s, *a);
        hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(PLAN_T), 0, s, *a);
    }
    hipLaunchKernelGGL(fork_apply_kernel, dim3(a->n_out, a->num_layers * 2), dim3(256), 0, s, *a);
    return (int)hipGetLastError();
}

extern "C" int g3k_pages_compact(const g3k_pages_args *a, void *stream) {
    hipStream_t s = (hipStream_t)stream;
    if (a->num_pages <= SMALL_PAGES && a->n_in <= SMALL_SEQS) {
        hipLaunchKernelGGL(compact_small_kernel, dim3(1), dim3(PLAN_T), 0, s, *a);
    } else {
        hipLaunchKernelGGL(pages_clear_kernel, dim3((a->num_pages + 255) / 256), dim3(256), 0, s, *a);
        hipLaunchKernelGGL(compact_count_kernel, dim3((a->n_in + 3) / 4), dim3(256), 0, s, *a);
        hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(PLAN_T), 0, s, *a);
    }
    hipLaunchKernelGGL(compact_apply_kernel, dim3(a->n_in + a->copy_wgs), dim3(256), 0, s, *a);
    return (int)hipGetLastError();
}
