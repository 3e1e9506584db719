// What the kernels of the paged cache share (gfx950).
#pragma once

#include <hip/hip_runtime.h>

#include "attn_common.h"
#include "paged_index.h"

namespace slm {

// paged_row for a row that is the wave's (every lane of it is active): up to 63
// sequences take one load of the starts and a ballot.
__device__ __forceinline__ PagedRow paged_row_wave(const PagedView& b, int row) {
    if (!b.row_start || b.n_seqs >= 64) return paged_row(b, row);
    const int lane = threadIdx.x & 63;
    const int start = b.row_start[min(lane, b.n_seqs)];
    const int below = __popcll(__ballot(lane <= b.n_seqs && start <= row));
    if (below == 0 || below > b.n_seqs) return PagedRow{-1, -1, false};
    const int end = min(__builtin_amdgcn_readlane(start, below), b.n_rows);
    if (row >= end) return PagedRow{-1, -1, false};  // starts that do not ascend
    return paged_row_of(b, below - 1, end, row);
}

// Sum over the lanes up to this one, in DPP steps: within the 16-lane rows, then
// the last lane of a row to the next, then that of the first two to the others.
__device__ __forceinline__ int wave_upto(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);  // row_shr:2
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);  // row_shr:4
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);  // row_shr:8
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast:15
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast:31
    return x;
}

__device__ __forceinline__ int wave_total(int x) {
    return __builtin_amdgcn_readlane(wave_upto(x), 63);
}

}  // namespace slm
