/*
 * slm_paged -- a paged KV cache of many sequences, and the attention over it.
 *
 * static-lm answers one sequence, whose cache rows lie one after another in
 * the arena (slm_attn.h).  A program that serves several at once keeps their
 * rows in pages of a common pool instead: a sequence takes pages as it grows,
 * gives them back when it ends, and sequences that begin alike may share
 * pages.  The entry points here have no counterpart in the reference; each
 * stands for the call of slm_attn.h that it widens:
 *   slm_paged_append_dev  slm_kv_append_dev and slm_rope_apply_dev, with
 *                         optional norms of the q and k heads in the same pass
 *   slm_paged_attend_dev  slm_attn_attend_dev (one new token per sequence) and
 *                         slm_attn_attend_batch_dev (runs of new rows), with
 *                         an optional window and first rows that stay visible
 * Conventions, error codes and streams are those of slm_attn.h; *_dev calls
 * take 16-byte-aligned device pointers (the int32 arrays of a batch: 4-byte
 * aligned) and are enqueued on the context's stream without waiting.  They
 * allocate nothing and can be captured into graphs.
 */
#ifndef SLM_PAGED_H
#define SLM_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "slm_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Types of a cache's values.  f32 rows hold what the arena's would, bit for
 * bit (without a head norm); bf16 halves the bytes, each value rounded once,
 * to nearest, when it is appended. */
enum { SLM_PAGED_F32 = 0, SLM_PAGED_BF16 = 1 };

typedef struct slm_paged_config {
    int32_t num_layers;
    int32_t num_pages;  /* of the pool, for each layer */
    int32_t page_size;  /* rows of a page: 16, 32, 64, 128 or 256 */
    int32_t dtype;      /* SLM_PAGED_F32 or SLM_PAGED_BF16 */
    int32_t max_seqs;   /* the most sequences of one call, 1 to 65536 */
} slm_paged_config;

typedef struct slm_paged_cache slm_paged_cache;

/* A cache for the heads and on the device of `ctx`, whose RoPE tables and
 * stream its calls use; only that context may be given with it.  The pool is
 * zeroed; it and the workspace for rows that are split over workgroups are the
 * cache's until slm_paged_destroy.  (The workspace has 65536 rows of head_dim + 2
 * floats, or num_heads * max_seqs + 8192 if that is more: 34 MB for 32 heads of
 * 128 and up to 1792 sequences.)  Calls and replayed graphs with one cache
 * share its rows and workspace: a program that moves its context to another
 * stream orders the two.  Destroy a cache when the work that uses it has
 * finished (slm_attn_sync), before or after the context's own destruction.
 * SLM_ERR_CONFIG for a value out of its range. */
int slm_paged_create(slm_attn_ctx* ctx, const slm_paged_config* cfg, slm_paged_cache** out);
void slm_paged_destroy(slm_paged_cache* cache);

/* The pool: [layer][page][K|V][kv head][row of page][head_dim] values of the
 * cache's type.  slm_paged_offset counts values from the base ((size_t)-1 for
 * an argument out of range).  For programs that move, copy or save pages. */
void* slm_paged_device_ptr(const slm_paged_cache* cache);
size_t slm_paged_offset(const slm_paged_cache* cache, int32_t layer, int32_t page, int32_t which,
                        int32_t kv_head, int32_t row);

/* What a call works on.  The arrays lie on the device and are read when the
 * kernels run, so a replayed graph sees their new values; the other fields
 * are read by the call.
 *
 * Sequence s holds lens[s] rows, its new ones included; row t of it is row t %
 * page_size of page page_table[s * table_stride + t / page_size].  Row r of q
 * (k, v, out), row_start[s] <= r < row_start[s + 1], is one of the sequence's
 * new rows, and its last rows' positions are theirs: row row_start[s + 1] - 1
 * sits at position lens[s] - 1.  Without row_start there is one row per
 * sequence (row s for sequence s): the form for single tokens.
 *
 *   - A sequence may have no new rows, and row_start[n_seqs] may lie below
 *     n_rows: rows that belong to no sequence are neither read nor written.
 *   - A row whose position would be negative (lens[s] = 0 in a batch rounded
 *     up with empty sequences) appends nothing and attends to nothing: its
 *     output is zeros.
 *   - lens[s] outside 0..max_len, or a page id outside the pool: nothing is
 *     read or written there, and the output rows that needed it are NaN
 *     (append: q_out for a bad length, nothing for a bad page).
 *   - Page ids of rows that no call reads or writes need not be valid, and
 *     what lies in a page behind the sequence's end is never used. */
typedef struct slm_paged_batch {
    int32_t n_seqs;       /* 0: the call does nothing */
    int32_t n_rows;       /* rows of q, k, v and out; n_seqs without row_start */
    int32_t max_len;      /* no sequence is longer; at most max_seq_len and the
                           * table's table_stride * page_size rows.  A bound near
                           * the longest length spares workgroups; the results do
                           * not depend on it beyond rounding */
    int32_t table_stride; /* page ids per sequence */
    const int32_t* page_table; /* [n_seqs][table_stride] */
    const int32_t* lens;       /* [n_seqs] */
    const int32_t* row_start;  /* [n_seqs + 1], ascending, or NULL */
} slm_paged_batch;

/* For every row r of the batch, at position p: each head of q [n_rows][dim]
 * and k [n_rows][kv_dim] is multiplied by 1 / sqrt(mean(x^2) + norm_eps) and
 * by q_norm / k_norm [head_dim] (f32; either may be NULL: no norm), then
 * rotated with the tables' row p.  q goes to q_out (q itself, or apart from
 * it), k and v [n_rows][kv_dim] to the sequence's page.  q and q_out may both
 * be NULL.  Without norms the arithmetic is slm_kv_append_dev's, and f32 pages
 * and q_out get its bits.  Rows of one call must go to different cache rows: a
 * page that two sequences share may be read by both, and appended to by one
 * of them in a call (else each value is one of those written). */
int slm_paged_append_dev(slm_attn_ctx* ctx, slm_paged_cache* cache, int32_t layer,
                         const slm_paged_batch* batch, const float* q, const float* k,
                         const float* v, const float* q_norm, const float* k_norm,
                         float norm_eps, float* q_out);

/* Attention of rotated q rows [n_rows][dim] over their sequences' pages: row r
 * at position p sees the rows t <= p (its own was appended before), and with
 * window > 0 of those only t > p - window and t < sinks.  window 0: all, and
 * sinks has no effect.  Scores are q . k / sqrt(head_dim); all sums and the
 * softmax are in f32.  A sequence's result depends on the other sequences of
 * the call by rounding only (they decide where its rows are split); the same
 * batch gives the same bits.  Visible rows of K must be finite.  K values
 * of bf16 pages below 2^-90 may lose digits, or count as 0. */
int slm_paged_attend_dev(slm_attn_ctx* ctx, slm_paged_cache* cache, int32_t layer,
                         const slm_paged_batch* batch, const float* q_rot, int32_t window,
                         int32_t sinks, float* out);

#ifdef __cplusplus
}
#endif

#endif /* SLM_PAGED_H */
