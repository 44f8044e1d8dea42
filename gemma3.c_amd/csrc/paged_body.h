// paged_body.h - what the kernels of the paged KV cache share: lengths and
// packed rows of a batch's sequences, read from device memory and kept within
// the buffers whatever they hold, and integer reductions over a wave.
#ifndef G3K_PAGED_BODY_H
#define G3K_PAGED_BODY_H

#include "g3k.h"
#include "g3k_device.h"

namespace g3k {

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }

__device__ __forceinline__ int wave_sum_int(int v) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m);
    return v;
}

// Sum over lanes 0..l.
__device__ __forceinline__ int wave_scan_int(int v, int lane) {
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const int o = __shfl(v, lane >= m ? lane - m : lane);
        v += lane >= m ? o : 0;
    }
    return v;
}

__device__ __forceinline__ int row16_min_int(int v) {
#pragma unroll
    for (int m = 1; m < 16; m *= 2) v = min(v, __shfl_xor(v, m));
    return v;
}

// The length of sequence b, within its table.
__device__ __forceinline__ int seq_len(const g3k_paged_seqs &s, int b) {
    return clampi(s.kv_len[b], 0, s.table_stride << s.page_shift);
}

// Packed rows of sequence b: the first, and how many.
__device__ __forceinline__ void seq_rows(const g3k_paged_seqs &s, int b, int &first, int &n) {
    if (!s.q_start) {
        first = b;
        n = 1;
        return;
    }
    first = clampi(s.q_start[b], 0, s.total_q);
    n = clampi(s.q_start[b + 1], first, s.total_q) - first;
}

}  // namespace g3k

#endif
