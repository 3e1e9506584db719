// Where the rows of a batch lie in a paged cache: every index that a kernel
// forms from a batch's device arrays, which may hold anything.  No HIP
// dependencies, so host code and CPU tests can include it as well as the
// kernels.
#pragma once

#include <stddef.h>
#include <stdint.h>

#if defined(__HIPCC__)
#define SLM_HD __host__ __device__ __forceinline__
#else
#define SLM_HD inline
#endif

namespace slm {

constexpr int kPagedMaxSeqs = 65536;

SLM_HD int paged_min(int a, int b) { return a < b ? a : b; }
SLM_HD int paged_max(int a, int b) { return a < b ? b : a; }

// A batch (slm_paged_batch) over one layer's pages [page][K|V][kv
// head][row][head_dim].  Every index that comes from device memory is checked
// before it is used: lengths against max_len, row ranges against n_rows, page
// ids against num_pages.
struct PagedView {
    void* pages;
    const int32_t* table;
    const int32_t* lens;
    const int32_t* row_start;  // nullptr: row s belongs to sequence s
    int n_seqs;
    int n_rows;
    int max_len;
    int stride;
    int num_pages;
    int ps_shift;   // log2 of the rows of a page
    int kv_heads;
};

// A row of the batch: its sequence and its position in it.
struct PagedRow {
    int seq;      // -1: the row belongs to no sequence
    int pos;      // < 0: an empty row
    bool bad;     // the sequence's length is out of range
};

// Row `row` of sequence seq, whose rows end before row `end` (> row).
SLM_HD PagedRow paged_row_of(const PagedView& b, int seq, int end, int row) {
    const int len = b.lens[seq];
    const bool bad = len < 0 || len > b.max_len;
    return PagedRow{seq, bad ? -1 : len - (end - row), bad};
}

// The row's sequence, found by one thread for itself: a binary search for the
// last row_start at or below the row.  (With sequences that have no rows
// several starts are equal; the last of them has the row.)
SLM_HD PagedRow paged_row(const PagedView& b, int row) {
    if (!b.row_start) return paged_row_of(b, row, row + 1, row);
    int lo = 0, hi = b.n_seqs;  // row_start[lo] <= row < row_start[hi], were they sentinels
    if (row < b.row_start[0] || row >= b.row_start[b.n_seqs]) return PagedRow{-1, -1, false};
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (b.row_start[mid] <= row)
            lo = mid;
        else
            hi = mid;
    }
    const int end = paged_min(b.row_start[lo + 1], b.n_rows);
    if (row >= end) return PagedRow{-1, -1, false};  // starts that do not ascend
    return paged_row_of(b, lo, end, row);
}

SLM_HD bool paged_page_ok(const PagedView& b, int page) { return page >= 0 && page < b.num_pages; }

// Values from the layer's base to row `slot` of K (which 0) or V (1) of a page
// and head; a pool may hold more than 2^31 of them.
SLM_HD size_t paged_at(const PagedView& b, int page, int which, int g, int slot, int hd) {
    return (((((size_t)page * 2 + which) * b.kv_heads + g) << b.ps_shift) + slot) * hd;
}

// Rows t that position p sees: all t <= p, or with a window the last `window`
// of them and the first `sinks`.  They are numbered u = 0 .. count - 1 without
// the gap: row(u).
struct Visible {
    int first;  // sinks in front of the gap
    int lo;     // first row behind it
    int count;
    SLM_HD Visible(int pos, int window, int sinks) {
        lo = window > 0 ? paged_max(0, pos + 1 - window) : 0;
        first = paged_min(sinks, lo);
        count = pos < 0 ? 0 : first + pos + 1 - lo;
    }
    SLM_HD int row(int u) const { return u < first ? u : u - first + lo; }
};

}  // namespace slm

#undef SLM_HD
