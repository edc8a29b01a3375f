// The paged K/V cache: page tables of a step, rows into pages and back, attention over them.
#include <math.h>

#include <algorithm>
#include <new>

#include "internal.h"

using namespace qimm_host;

struct qimm_pages {
    qimm_ctx *ctx = nullptr;
    int64_t layers = 0;
    qimm::PageDims dims{};
    uint8_t *mem = nullptr;
    void *scratch = nullptr;  // of the attention: its shares' sums
    uint8_t *layer(int64_t i) const { return mem + i * dims.layer_bytes(); }
    int64_t cache_bytes() const { return layers * dims.layer_bytes(); }
    int64_t scratch_bytes() const { return (int64_t)qimm::paged_attention_scratch(dims.head_dim); }
};

namespace {

constexpr int64_t MAX_TOKENS = (int64_t)1 << 31;  // slots and granules are int32
constexpr int64_t MAX_REQUESTS = 65536;
constexpr int64_t MAX_ROWS = (int64_t)1 << 28;     // of a store, 16 a workgroup

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

bool page_size_fits(int64_t page_size) { return page_size >= 16 && page_size <= 512 && page_size % 16 == 0; }

int check_layer(const qimm_pages *pg, int64_t layer, const char *what) {
    if (layer < 0 || layer >= pg->layers) return set_err(pg->ctx, QIMM_ERR_SHAPE, std::string(what) + ": layer out of range");
    return QIMM_OK;
}

}  // namespace

extern "C" {

int qimm_page_plan(qimm_ctx *ctx, const qimm_page_plan_args *p, void *stream) {
    if (!ctx || !p) return QIMM_ERR_ARG;
    if (!page_size_fits(p->page_size))
        return set_err(ctx, QIMM_ERR_SHAPE, "page plan: the page size must be a multiple of 16 up to 512");
    if (p->pages <= 0 || p->pages >= MAX_TOKENS / p->page_size)
        return set_err(ctx, QIMM_ERR_SHAPE, "page plan: 1 to 2^31 / page_size pages");
    if (p->requests <= 0 || p->requests > MAX_REQUESTS) return set_err(ctx, QIMM_ERR_SHAPE, "page plan: 1 to 65536 requests");
    if (p->max_pages < 0 || p->max_pages >= MAX_TOKENS || p->max_rows < 0 || p->max_rows >= MAX_TOKENS)
        return set_err(ctx, QIMM_ERR_SHAPE, "page plan: bad sizes");
    if (!p->lengths || !p->added || !p->queue || !p->state || !p->lengths_out || !p->state_out || !p->starts || !p->work ||
        (p->max_pages && !p->tables) || (p->max_rows && !p->slots))
        return set_err(ctx, QIMM_ERR_ARG, "page plan: null array");
    QIMM_HIP(ctx, hipSetDevice(ctx->device));
    const qimm::PagePlanArgs a{p->pages, p->requests, p->max_pages, p->max_rows, (int)p->page_size, p->tables,
                               p->lengths, p->added, p->queue, p->state, p->lengths_out, p->state_out, p->starts,
                               p->slots, p->positions, p->work};
    QIMM_HIP(ctx, qimm::launch_page_plan(a, (hipStream_t)stream));
    return QIMM_OK;
}

int64_t qimm_page_plan_work(int64_t requests) {
    return requests <= 0 || requests > MAX_REQUESTS ? -1 : qimm::page_plan_work(requests);
}

int qimm_pages_create(qimm_ctx *ctx, int64_t layers, int64_t pages, int64_t page_size, int64_t kv_heads, int64_t head_dim,
                      qimm_pages **out) {
    if (!ctx || !out) return QIMM_ERR_ARG;
    *out = nullptr;
    if (head_dim != 64 && head_dim != 128) return set_err(ctx, QIMM_ERR_SHAPE, "pages: head_dim must be 64 or 128");
    if (!page_size_fits(page_size)) return set_err(ctx, QIMM_ERR_SHAPE, "pages: the page size must be a multiple of 16 up to 512");
    if (layers <= 0 || pages <= 0 || kv_heads <= 0 || kv_heads > 65535)
        return set_err(ctx, QIMM_ERR_SHAPE, "pages: layers and pages must be positive, 1 to 65535 heads");
    if (pages >= MAX_TOKENS / page_size || pages >= MAX_TOKENS / 2 / (kv_heads * (page_size / 16)))
        return set_err(ctx, QIMM_ERR_SHAPE, "pages: pages * page_size must be below 2^31, pages * kv_heads * page_size / 16 below 2^30");
    qimm_pages *pg = new (std::nothrow) qimm_pages();
    if (!pg) return set_err(ctx, QIMM_ERR_OOM, "pages: host allocation failed");
    pg->ctx = ctx;
    pg->layers = layers;
    pg->dims = qimm::PageDims{pages, (int)page_size, (int)kv_heads, (int)head_dim};
    if (layers > ((int64_t)1 << 60) / pg->dims.layer_bytes()) {
        delete pg;
        return set_err(ctx, QIMM_ERR_OOM, "pages: too large");
    }
    hipError_t e = hipSetDevice(ctx->device);
    if (e == hipSuccess) e = hipMalloc((void **)&pg->mem, (size_t)pg->cache_bytes());
    if (e == hipSuccess) e = hipMalloc(&pg->scratch, (size_t)pg->scratch_bytes());
    // the null stream does not order a later call on a non-blocking stream: wait for the fill
    if (e == hipSuccess) e = hipMemset(pg->scratch, 0, qimm::PAGED_COUNTER_BYTES);
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        if (pg->mem) (void)hipFree(pg->mem);
        if (pg->scratch) (void)hipFree(pg->scratch);
        delete pg;
        return hip_err(ctx, e, "hipMalloc(pages)");
    }
    *out = pg;
    return QIMM_OK;
}

int qimm_pages_destroy(qimm_pages *pg) {
    if (!pg) return QIMM_ERR_ARG;
    if (pg->mem) (void)hipFree(pg->mem);
    if (pg->scratch) (void)hipFree(pg->scratch);
    delete pg;
    return QIMM_OK;
}

int64_t qimm_pages_device_bytes(const qimm_pages *pg) { return pg ? pg->cache_bytes() + pg->scratch_bytes() : -1; }

int qimm_pages_store(qimm_pages *pg, int64_t layer, const void *k, const void *v, int type, int64_t rows, int64_t k_row,
                     int64_t k_head, int64_t v_row, int64_t v_head, const int32_t *slots, void *stream) {
    if (!pg || rows < 0 || (rows && (!k || !v || !slots))) return QIMM_ERR_ARG;
    qimm_ctx *ctx = pg->ctx;
    const int rc = check_layer(pg, layer, "pages store");
    if (rc) return rc;
    if (type != QIMM_TYPE_F32 && type != QIMM_TYPE_F16 && type != QIMM_TYPE_BF16)
        return set_err(ctx, QIMM_ERR_TYPE, "pages store: rows must be F32, F16 or BF16");
    const int64_t d = pg->dims.head_dim, unit = type == QIMM_TYPE_F32 ? 4 : 8;
    if (k_row < 0 || k_head < 0 || v_row < 0 || v_head < 0 || (k_row | k_head | v_row | v_head) % unit || !aligned16(k) ||
        !aligned16(v))
        return set_err(ctx, QIMM_ERR_ARG, "pages store: k, v and their strides must be 16-byte aligned");
    if (rows >= MAX_ROWS) return set_err(ctx, QIMM_ERR_SHAPE, "pages store: rows must be below 2^28");
    QIMM_HIP(ctx, hipSetDevice(ctx->device));
    const int64_t dense = pg->dims.kv_heads * d;
    QIMM_HIP(ctx, qimm::launch_pages_store(pg->dims, pg->layer(layer), k, v, type, k_row ? k_row : dense, k_head ? k_head : d,
                                           v_row ? v_row : dense, v_head ? v_head : d, slots, rows, (hipStream_t)stream));
    return QIMM_OK;
}

int qimm_pages_load(const qimm_pages *pg, int64_t layer, uint16_t *k, uint16_t *v, int64_t rows, const int32_t *slots,
                    void *stream) {
    if (!pg || rows < 0 || (rows && (!k || !v || !slots))) return QIMM_ERR_ARG;
    qimm_ctx *ctx = pg->ctx;
    const int rc = check_layer(pg, layer, "pages load");
    if (rc) return rc;
    if (!aligned16(k) || !aligned16(v)) return set_err(ctx, QIMM_ERR_ARG, "pages load: k and v must be 16-byte aligned");
    if (rows >= MAX_ROWS) return set_err(ctx, QIMM_ERR_SHAPE, "pages load: rows must be below 2^28");
    QIMM_HIP(ctx, hipSetDevice(ctx->device));
    QIMM_HIP(ctx, qimm::launch_pages_load(pg->dims, pg->layer(layer), k, v, slots, rows, (hipStream_t)stream));
    return QIMM_OK;
}

int qimm_attention_paged(qimm_pages *pg, int64_t layer, const qimm_paged_attention *x, void *stream) {
    if (!pg || !x) return QIMM_ERR_ARG;
    qimm_ctx *ctx = pg->ctx;
    const int rc = check_layer(pg, layer, "paged attention");
    if (rc) return rc;
    const int64_t d = pg->dims.head_dim;
    if (x->rows < 0 || x->requests < 0 || x->requests > MAX_REQUESTS || x->max_pages < 0 || x->heads <= 0)
        return set_err(ctx, QIMM_ERR_SHAPE, "paged attention: bad sizes (at most 65536 requests)");
    if (x->heads % pg->dims.kv_heads) return set_err(ctx, QIMM_ERR_SHAPE, "paged attention: heads must be a multiple of the cache's");
    if (!x->starts && x->rows != x->requests)
        return set_err(ctx, QIMM_ERR_SHAPE, "paged attention: without starts every request has one row");
    if (x->rows >= (MAX_TOKENS - 64) / x->heads) return set_err(ctx, QIMM_ERR_SHAPE, "paged attention: rows * heads must be below 2^31 - 64");
    // the grid of the attention: tiles of 128 rows and heads, one more a request, and the shares
    if (x->rows * x->heads / 128 + std::min(x->requests, x->rows) * pg->dims.kv_heads * 2 >= ((int64_t)1 << 24) - 8192)
        return set_err(ctx, QIMM_ERR_SHAPE, "paged attention: too many rows and requests for one call");
    if (x->window < 0 || x->sinks < 0 || (x->window && !x->causal) || (x->sinks && !x->window))
        return set_err(ctx, QIMM_ERR_ARG, "paged attention: a window needs causal rows, sinks a window");
    if (!isfinite(x->scale) || x->scale <= 0.f) return set_err(ctx, QIMM_ERR_ARG, "paged attention: the scale must be positive and finite");
    if (x->rows == 0 || x->requests == 0) return QIMM_OK;
    if (!x->q || !x->out || !x->lengths || (x->max_pages && !x->tables)) return set_err(ctx, QIMM_ERR_ARG, "paged attention: null array");
    if (!aligned16(x->q) || !aligned16(x->out) || x->q_row < 0 || x->q_head < 0 || (x->q_row | x->q_head) % 8)
        return set_err(ctx, QIMM_ERR_ARG, "paged attention: q, its strides and out must be 16-byte aligned");
    QIMM_HIP(ctx, hipSetDevice(ctx->device));
    const qimm::PagedAttnArgs a{x->q, x->q_row ? x->q_row : x->heads * d, x->q_head ? x->q_head : d, x->rows, x->heads,
                                x->tables, x->requests, x->max_pages, x->lengths, x->starts, x->causal, x->window,
                                x->sinks, x->scale, x->out};
    QIMM_HIP(ctx, qimm::launch_paged_attention(pg->dims, pg->layer(layer), a, pg->scratch, (hipStream_t)stream));
    return QIMM_OK;
}

}  // extern "C"
