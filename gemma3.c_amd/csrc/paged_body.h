// paged_body.h - what the kernels of the paged KV cache share: lengths and
// packed rows of a batch's sequences, read from device memory and kept within
// the buffers whatever they hold, and integer reductions over a wave.
#ifndef G3K_PAGED_BODY_H
#define G3K_PAGED_BODY_H

#include "g3k.h"
#include "g3k_device.h"

namespace g3k {

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }


// Sum over lanes 0..l: within rows of 16 lanes, then the rows' totals.
__device__ __forceinline__ int wave_scan_int(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);    // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row_bcast:15 to rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // row_bcast:31 to rows 2 and 3
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

__device__ __forceinline__ int wave_sum_int(int v) { return __builtin_amdgcn_readlane(wave_scan_int(v), 63); }

}  // namespace g3k

#endif
