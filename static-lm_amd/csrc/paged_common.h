// What the kernels of the paged cache share (gfx950).
#pragma once

#include <hip/hip_runtime.h>

#include "attn_common.h"
#include "paged_index.h"

namespace slm {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));

// Two values as bf16 pairs: x = p1 + p2 + p3 (24 bits).
__device__ __forceinline__ void split2(float x0, float x1, uint32_t* p1, uint32_t* p2,
                                       uint32_t* p3) {
    const auto pack = [](float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{a, b}, bf2));
    };
    *p1 = pack(x0, x1);
    x0 -= __uint_as_float(*p1 << 16);
    x1 -= __uint_as_float(*p1 & 0xFFFF0000u);
    *p2 = pack(x0, x1);
    x0 -= __uint_as_float(*p2 << 16);
    x1 -= __uint_as_float(*p2 & 0xFFFF0000u);
    *p3 = pack(x0, x1);
}

__device__ __forceinline__ void split8(const float* x, bf8 (&p)[3]) {
    u4 w[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t a, b, c;
        split2(x[2 * i], x[2 * i + 1], &a, &b, &c);
        w[0][i] = a, w[1][i] = b, w[2][i] = c;
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) p[k] = __builtin_bit_cast(bf8, w[k]);
}

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
