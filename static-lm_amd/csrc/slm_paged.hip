// Host side of slm_paged.h: the paged cache's handle, the checks of its calls
// and their dispatch.
#include "../../include/slm_paged.h"

#include <limits.h>
#include <stdint.h>

#include <new>
#include <string>

#include "paged_common.h"
#include "slm_host.h"

struct slm_paged_cache {
    const slm_attn_ctx* ctx = nullptr;  // compared only: the context may be gone
    slm_paged_config cfg{};
    int device = 0;
    int num_heads = 0, kv_heads = 0, head_dim = 0;
    int ps_shift = 0;
    void* pool = nullptr;
    size_t layer_bytes = 0;
    // partial results of split rows and tiles
    float* part_o = nullptr;
    float* part_ml = nullptr;
};

using namespace slm_host;

namespace {

size_t value_bytes(const slm_paged_cache* c) { return c->cfg.dtype == SLM_PAGED_BF16 ? 2 : 4; }

size_t pool_bytes(const slm_paged_cache* c) { return c->layer_bytes * c->cfg.num_layers; }

// Lets go of what a cache holds on its device, whichever is current.
void release(slm_paged_cache* c) {
    int prev = -1;
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    if (prev != c->device) (void)hipSetDevice(c->device);
    (void)hipFree(c->pool);
    (void)hipFree(c->part_o);
    (void)hipFree(c->part_ml);
    if (prev >= 0 && prev != c->device) (void)hipSetDevice(prev);
    delete c;
}

// The context's device is current while a call launches on its stream.
struct OnDevice {
    int prev = -1;
    explicit OnDevice(int device) {
        int d = -1;
        if (hipGetDevice(&d) == hipSuccess && d != device && hipSetDevice(device) == hipSuccess)
            prev = d;
    }
    ~OnDevice() {
        if (prev >= 0) (void)hipSetDevice(prev);
    }
};

// The checks that the two calls share.
int check_call(slm_attn_ctx* c, const slm_paged_cache* cache, int layer,
               const slm_paged_batch* b) {
    if (!cache || !b) return fail(c, SLM_ERR_ARG, "cache or batch is NULL");
    // (the heads too: a new context may lie where the cache's own one did)
    const slm::Shape& s = c->shape;
    if (cache->ctx != c || cache->device != c->device || cache->num_heads != s.num_heads ||
        cache->kv_heads != s.num_kv_heads || cache->head_dim != s.head_dim)
        return fail(c, SLM_ERR_ARG, "the cache belongs to another context");
    if (layer < 0 || layer >= cache->cfg.num_layers)
        return fail(c, SLM_ERR_LAYER, "layer index out of range");
    if (b->n_seqs < 0 || b->n_rows < 0)
        return fail(c, SLM_ERR_BATCH, "n_seqs and n_rows must not be negative");
    if (b->n_seqs > cache->cfg.max_seqs)
        return fail(c, SLM_ERR_BATCH, "more sequences than the cache's max_seqs");
    if (b->n_seqs == 0 || b->n_rows == 0) return SLM_OK;
    if (!b->row_start && b->n_rows != b->n_seqs)
        return fail(c, SLM_ERR_BATCH, "without row_start there is one row per sequence");
    if (!b->page_table || !b->lens) return fail(c, SLM_ERR_ARG, "NULL buffer");
    for (const int32_t* p : {b->page_table, b->lens, b->row_start})
        if ((uintptr_t)p & 3u) return fail(c, SLM_ERR_ARG, "int32 arrays must be 4-byte aligned");
    if (b->table_stride <= 0) return fail(c, SLM_ERR_BATCH, "table_stride must be positive");
    if (b->max_len <= 0 || b->max_len > c->cfg.max_seq_len ||
        b->max_len > (int64_t)b->table_stride * cache->cfg.page_size)
        return fail(c, SLM_ERR_BATCH,
                    "max_len must be positive and at most max_seq_len and the table's rows");
    // workgroups of 256 threads are counted in 24 bits
    if ((int64_t)b->n_rows * s.num_heads + (int64_t)b->n_seqs * s.num_kv_heads >= INT64_C(1) << 23)
        return fail(c, SLM_ERR_BATCH, "too many rows and heads in one call (2^23)");
    // the split decode adds up the sequences' tiles of 16 rows or more in 32 bits
    if ((int64_t)b->n_seqs * (b->max_len / 16 + 1) >= INT64_C(1) << 30)
        return fail(c, SLM_ERR_BATCH, "n_seqs * max_len must be below 2^34");
    return SLM_OK;
}

slm::PagedView view_of(const slm_paged_cache* cache, int layer, const slm_paged_batch* b) {
    return slm::PagedView{static_cast<char*>(cache->pool) + cache->layer_bytes * layer,
                          b->page_table,
                          b->lens,
                          b->row_start,
                          b->n_seqs,
                          b->n_rows,
                          b->max_len,
                          b->table_stride,
                          cache->cfg.num_pages,
                          cache->ps_shift,
                          cache->kv_heads};
}

// A buffer that a call writes must not overlap the pool or the batch's arrays.
int check_written(slm_attn_ctx* c, const slm_paged_cache* cache, const slm_paged_batch* b,
                  const void* p, size_t bytes, const char* name) {
    if (overlaps(p, bytes, cache->pool, pool_bytes(cache)) ||
        overlaps(p, bytes, b->page_table, (size_t)b->n_seqs * b->table_stride * 4) ||
        overlaps(p, bytes, b->lens, (size_t)b->n_seqs * 4) ||
        (b->row_start && overlaps(p, bytes, b->row_start, ((size_t)b->n_seqs + 1) * 4)))
        return fail(c, SLM_ERR_ALIAS,
                    std::string(name) + " must not overlap the cache or the batch's arrays");
    return SLM_OK;
}

}  // namespace

extern "C" {

int slm_paged_create(slm_attn_ctx* ctx, const slm_paged_config* cfg, slm_paged_cache** out) {
    if (!out) return fail(ctx, SLM_ERR_ARG, "out is NULL");
    *out = nullptr;
    if (!ctx) return fail(nullptr, SLM_ERR_ARG, "ctx is NULL");
    if (!cfg) return fail(ctx, SLM_ERR_ARG, "config is NULL");
    if (ctx->capturing) return refuse_capture(ctx, "slm_paged_create");
    if (cfg->num_layers <= 0 || cfg->num_pages <= 0)
        return fail(ctx, SLM_ERR_CONFIG, "num_layers and num_pages must be positive");
    if (cfg->page_size < 16 || cfg->page_size > 256 || (cfg->page_size & (cfg->page_size - 1)))
        return fail(ctx, SLM_ERR_CONFIG, "page_size must be 16, 32, 64, 128 or 256");
    if (cfg->dtype != SLM_PAGED_F32 && cfg->dtype != SLM_PAGED_BF16)
        return fail(ctx, SLM_ERR_CONFIG, "dtype must be SLM_PAGED_F32 or SLM_PAGED_BF16");
    if (cfg->max_seqs <= 0 || cfg->max_seqs > slm::kPagedMaxSeqs)
        return fail(ctx, SLM_ERR_CONFIG, "max_seqs must be 1 to 65536");
    const slm::Shape& s = ctx->shape;
    slm_paged_cache* c = new (std::nothrow) slm_paged_cache();
    if (!c) return fail(ctx, SLM_ERR_HIP, "out of host memory for the cache handle");
    c->ctx = ctx;
    c->cfg = *cfg;
    c->device = ctx->device;
    c->num_heads = s.num_heads;
    c->kv_heads = s.num_kv_heads;
    c->head_dim = s.head_dim;
    while ((1 << c->ps_shift) < cfg->page_size) ++c->ps_shift;
    const double want = (double)cfg->num_layers * cfg->num_pages * 2 * cfg->page_size * s.kv_dim *
                        value_bytes(c);
    if (want > (double)(INT64_C(1) << 46)) {
        delete c;
        return fail(ctx, SLM_ERR_CONFIG, "the pool would exceed 64 TiB");
    }
    c->layer_bytes = (size_t)cfg->num_pages * 2 * cfg->page_size * s.kv_dim * value_bytes(c);
    const size_t chunks = slm::paged_decode_chunks(s, cfg->max_seqs) * s.num_heads;
    const size_t rows = slm::paged_prefill_part_rows(s);
    const size_t parts = chunks > rows ? chunks : rows;
    int prev = -1;
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    hipError_t e = hipSetDevice(c->device);
    const char* what = "hipMalloc(paged cache)";
    if (e == hipSuccess) e = hipMalloc(&c->pool, pool_bytes(c));
    if (e == hipSuccess) e = hipMalloc(&c->part_o, parts * s.head_dim * sizeof(float));
    if (e == hipSuccess) e = hipMalloc(&c->part_ml, parts * 2 * sizeof(float));
    if (e == hipSuccess) {
        what = "hipMemset(paged cache)";
        e = hipMemset(c->pool, 0, pool_bytes(c));
    }
    // the memset runs on the default stream, the cache's calls on any other
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (prev >= 0) (void)hipSetDevice(prev);
    if (e != hipSuccess) {
        release(c);
        return hip_fail(ctx, e, what);
    }
    *out = c;
    return SLM_OK;
}

void slm_paged_destroy(slm_paged_cache* cache) {
    if (cache) release(cache);
}

void* slm_paged_device_ptr(const slm_paged_cache* cache) { return cache ? cache->pool : nullptr; }

size_t slm_paged_offset(const slm_paged_cache* c, int32_t layer, int32_t page, int32_t which,
                        int32_t kv_head, int32_t row) {
    if (!c || layer < 0 || layer >= c->cfg.num_layers || page < 0 || page >= c->cfg.num_pages ||
        (which != 0 && which != 1) || kv_head < 0 || kv_head >= c->kv_heads || row < 0 ||
        row >= c->cfg.page_size)
        return (size_t)-1;
    return (((((size_t)layer * c->cfg.num_pages + page) * 2 + which) * c->kv_heads + kv_head) *
                c->cfg.page_size +
            row) *
           c->head_dim;
}

int slm_paged_append_dev(slm_attn_ctx* c, slm_paged_cache* cache, int32_t layer,
                         const slm_paged_batch* b, const float* q, const float* k,
                         const float* v, const float* q_norm, const float* k_norm,
                         float norm_eps, float* q_out) {
    if (!c) return fail(nullptr, SLM_ERR_ARG, "ctx is NULL");
    int rc;
    if ((rc = check_call(c, cache, layer, b))) return rc;
    if (!(norm_eps >= 0.0f) && (q_norm || k_norm))
        return fail(c, SLM_ERR_ARG, "norm_eps must not be negative");
    if ((q == nullptr) != (q_out == nullptr))
        return fail(c, SLM_ERR_ARG, "q and q_out go together");
    if (b->n_seqs == 0 || b->n_rows == 0) return SLM_OK;
    const slm::Shape& s = c->shape;
    if ((rc = check_dev_ptrs(c, {k, v})) || (q && (rc = check_dev_ptrs(c, {q, q_out}))) ||
        (q_norm && (rc = check_dev_ptrs(c, {q_norm}))) ||
        (k_norm && (rc = check_dev_ptrs(c, {k_norm}))))
        return rc;
    const size_t qb = (size_t)b->n_rows * s.dim * 4, kb = (size_t)b->n_rows * s.kv_dim * 4;
    const size_t wb = (size_t)s.head_dim * 4;
    if (overlaps(k, kb, cache->pool, pool_bytes(cache)) ||
        overlaps(v, kb, cache->pool, pool_bytes(cache)) ||
        (q && overlaps(q, qb, cache->pool, pool_bytes(cache))))
        return fail(c, SLM_ERR_ALIAS, "q, k and v must not overlap the cache");
    if (q) {
        if ((rc = check_written(c, cache, b, q_out, qb, "q_out"))) return rc;
        if ((q_out != q && overlaps(q_out, qb, q, qb)) || overlaps(q_out, qb, k, kb) ||
            overlaps(q_out, qb, v, kb) || (q_norm && overlaps(q_out, qb, q_norm, wb)) ||
            (k_norm && overlaps(q_out, qb, k_norm, wb)))
            return fail(c, SLM_ERR_ALIAS,
                        "q_out must be q itself or overlap no input of the call");
    }
    const slm::PagedView view = view_of(cache, layer, b);
    const OnDevice on(c->device);
    Timed t(c, SLM_K_APPEND);
    const hipError_t e = slm::launch_paged_append(s, view, cache->cfg.dtype == SLM_PAGED_BF16, q, k,
                                                  v, q_norm, k_norm, norm_eps, c->cos_t, c->sin_t,
                                                  q_out, c->stream);
    t.done();
    return launch_status(c, e, "paged append kernel launch");
}

int slm_paged_attend_dev(slm_attn_ctx* c, slm_paged_cache* cache, int32_t layer,
                         const slm_paged_batch* b, const float* q_rot, int32_t window,
                         int32_t sinks, float* out) {
    if (!c) return fail(nullptr, SLM_ERR_ARG, "ctx is NULL");
    int rc;
    if ((rc = check_call(c, cache, layer, b))) return rc;
    if (window < 0 || sinks < 0)
        return fail(c, SLM_ERR_ARG, "window and sinks must not be negative");
    if (b->n_seqs == 0 || b->n_rows == 0) return SLM_OK;
    if ((rc = check_dev_ptrs(c, {q_rot, out}))) return rc;
    const slm::Shape& s = c->shape;
    const size_t qb = (size_t)b->n_rows * s.dim * 4;
    if (overlaps(out, qb, q_rot, qb)) return fail(c, SLM_ERR_ALIAS, "out must not overlap q");
    if ((rc = check_written(c, cache, b, out, qb, "out"))) return rc;
    // a window that hides nothing from any row is none (and the kernels' sums of
    // positions and windows stay within 32 bits)
    if ((int64_t)window + sinks >= b->max_len) window = 0;
    const slm::PagedView view = view_of(cache, layer, b);
    const OnDevice on(c->device);
    const bool bf16 = cache->cfg.dtype == SLM_PAGED_BF16;
    if (b->row_start) {
        Timed t(c, SLM_K_PREFILL);
        const hipError_t e =
            slm::launch_paged_prefill(s, view, bf16, q_rot, window, sinks, cache->part_o,
                                      cache->part_ml, out, c->stream);
        t.done();
        return launch_status(c, e, "paged prefill kernel launch");
    }
    Timed t(c, SLM_K_DECODE);
    const hipError_t e = slm::launch_paged_decode(s, view, bf16, q_rot, window, sinks,
                                                  cache->part_o, cache->part_ml, out, c->stream);
    t.done();
    return launch_status(c, e, "paged decode kernel launch");
}

}  // extern "C"
