// Low-rank adapters of many requests beside a quantized projection.
#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

#include "internal.h"

using namespace qimm_host;

struct qimm_adapters {
    qimm_ctx *ctx = nullptr;
    int64_t rows = 0, cols = 0, count = 0, max_rank = 0;
    void *dev = nullptr;                // the table of AdapterDev, then every A and B
    size_t bytes = 0;
    const qimm::AdapterDev *table() const { return (const qimm::AdapterDev *)dev; }
    int64_t ldt() const { return (max_rank + 31) / 32 * 32; }
};

namespace {

size_t align_up(size_t v) { return (v + 255) & ~(size_t)255; }

// Scratch of one product in the context's growable workspace: t, and for bf16 outputs the
// f32 sums.
struct Scratch {
    size_t base, total;
};
Scratch scratch_of(const qimm_adapters *ad, int64_t m, int out_type) {
    Scratch s{};
    s.base = align_up((size_t)(m * ad->ldt()) * 4);
    s.total = s.base + (out_type == QIMM_TYPE_F32 ? 0 : (size_t)(m * ad->rows) * 4);
    return s;
}

int check_pair(qimm_ctx *ctx, const qimm_weight *w, const qimm_adapters *ad) {
    if (ad->rows != w->rows || ad->cols != w->cols)
        return set_err(ctx, QIMM_ERR_SHAPE, "qmatmul with adapters: the adapters' rows x cols differ from the weight's");
    if (w->ctx->device != ctx->device || ad->ctx->device != ctx->device)
        return set_err(ctx, QIMM_ERR_STATE, "qmatmul with adapters: weight or adapters live on another device");
    return QIMM_OK;
}

int reserve(qimm_ctx *ctx, const qimm_weight *w, const qimm_adapters *ad, int64_t m, int out_type) {
    QIMM_HIP(ctx, hipSetDevice(ctx->device));
    if (const int rc = ensure_workspace(ctx, scratch_of(ad, m, out_type).total)) return rc;
    if (const size_t need = qimm::qgemm_workspace(w->gw, m))
        if (const int rc = ensure_part_workspace(ctx, need)) return rc;
    return QIMM_OK;
}

}  // namespace

extern "C" {

int qimm_adapters_create(qimm_ctx *ctx, int64_t rows, int64_t cols, const qimm_adapter *list, int64_t n,
                         qimm_adapters **out) {
    if (!ctx || !out || n < 0 || (n > 0 && !list)) return QIMM_ERR_ARG;
    *out = nullptr;
    if (rows <= 0 || rows % 128 || cols <= 0 || cols % 64)
        return set_err(ctx, QIMM_ERR_SHAPE, "adapters: needs rows % 128 == 0 and cols % 64 == 0");
    if (n < 1 || n > 65535) return set_err(ctx, QIMM_ERR_SHAPE, "adapters: 1 to 65535 of them");
    for (int64_t i = 0; i < n; i++) {
        const qimm_tensor &a = list[i].a, &b = list[i].b;
        if (!a.data || !b.data) return set_err(ctx, QIMM_ERR_ARG, "adapters: missing tensor");
        if (a.ggml_type != b.ggml_type ||
            (a.ggml_type != QIMM_TYPE_F32 && a.ggml_type != QIMM_TYPE_F16 && a.ggml_type != QIMM_TYPE_BF16))
            return set_err(ctx, QIMM_ERR_TYPE, "adapters: a and b must both be F32, F16 or BF16");
        const int64_t r = a.rows, e = a.ggml_type == QIMM_TYPE_F32 ? 4 : 2;
        if (r < 1 || r > QIMM_ADAPTER_MAX_RANK || a.cols != cols || b.rows != rows || b.cols != r ||
            a.nbytes != (size_t)(r * cols * e) || b.nbytes != (size_t)(rows * r * e))
            return set_err(ctx, QIMM_ERR_SHAPE, "adapters: a must be [rank, cols] and b [rows, rank], rank 1 to " +
                                                    std::to_string(QIMM_ADAPTER_MAX_RANK));
    }
    qimm_adapters *ad = nullptr;
    try {
        ad = new qimm_adapters();
        ad->ctx = ctx;
        ad->rows = rows;
        ad->cols = cols;
        ad->count = n;
        std::vector<qimm::AdapterDev> table((size_t)n);
        std::vector<size_t> at_a((size_t)n), at_b((size_t)n);
        size_t off = align_up((size_t)n * sizeof(qimm::AdapterDev));
        for (int64_t i = 0; i < n; i++) {
            const int64_t r = list[i].a.rows, ldb = (r + 7) / 8 * 8;
            at_a[(size_t)i] = off;
            off += align_up((size_t)(r * cols) * 2);
            at_b[(size_t)i] = off;
            off += align_up((size_t)(rows * ldb) * 2);
            ad->max_rank = std::max(ad->max_rank, r);
        }
        ad->bytes = off;
        // A as it is; B's rows padded with zeros to 16 bytes
        std::vector<uint8_t> host(off, 0);
        for (int64_t i = 0; i < n; i++) {
            const int64_t r = list[i].a.rows, ldb = (r + 7) / 8 * 8;
            to_bf16(list[i].a.ggml_type, (const uint8_t *)list[i].a.data, r * cols, (uint16_t *)&host[at_a[(size_t)i]]);
            std::vector<uint16_t> b((size_t)(rows * r));
            to_bf16(list[i].b.ggml_type, (const uint8_t *)list[i].b.data, rows * r, b.data());
            for (int64_t row = 0; row < rows; row++)
                memcpy(&host[at_b[(size_t)i] + (size_t)(row * ldb) * 2], &b[(size_t)(row * r)], (size_t)r * 2);
        }
        hipError_t e = hipSetDevice(ctx->device);
        if (e == hipSuccess) e = hipMalloc(&ad->dev, off);
        if (e == hipSuccess) {
            for (int64_t i = 0; i < n; i++) {
                const int r = (int)list[i].a.rows;
                table[(size_t)i] = {(const uint16_t *)((char *)ad->dev + at_a[(size_t)i]),
                                    (const uint16_t *)((char *)ad->dev + at_b[(size_t)i]), r, (r + 7) / 8 * 8, list[i].scale, 0};
            }
            memcpy(host.data(), table.data(), table.size() * sizeof(qimm::AdapterDev));
            e = hipMemcpy(ad->dev, host.data(), off, hipMemcpyHostToDevice);
        }
        if (e != hipSuccess) {
            if (ad->dev) (void)hipFree(ad->dev);
            delete ad;
            return hip_err(ctx, e, "adapters upload");
        }
    } catch (const std::bad_alloc &) {
        delete ad;
        return set_err(ctx, QIMM_ERR_OOM, "adapters: host staging allocation failed");
    }
    *out = ad;
    return QIMM_OK;
}

int qimm_adapters_destroy(qimm_adapters *ad) {
    if (!ad) return QIMM_ERR_ARG;
    if (ad->dev) (void)hipFree(ad->dev);
    delete ad;
    return QIMM_OK;
}

int64_t qimm_adapters_device_bytes(const qimm_adapters *ad) { return ad ? (int64_t)ad->bytes : -1; }

int qimm_qmatmul_adapters_reserve(qimm_ctx *ctx, const qimm_weight *w, const qimm_adapters *ad, int64_t m, int out_type) {
    if (!ctx || !w || !ad || m < 0) return QIMM_ERR_ARG;
    if (out_type != QIMM_TYPE_F32 && out_type != QIMM_TYPE_BF16)
        return set_err(ctx, QIMM_ERR_TYPE, "qmatmul: output must be F32 or BF16");
    if (const int rc = check_pair(ctx, w, ad)) return rc;
    return reserve(ctx, w, ad, m, out_type);
}

int qimm_qmatmul_adapters(qimm_ctx *ctx, const qimm_weight *w, const qimm_adapters *ad, const int32_t *ids,
                          const void *x_bf16, int64_t m, int64_t lda, void *y, int out_type, void *stream) {
    if (!ad || !ids) return QIMM_ERR_ARG;
    if (const int rc = qmatmul_check(ctx, w, x_bf16, m, lda, y, out_type)) return rc;
    if (const int rc = check_pair(ctx, w, ad)) return rc;
    if ((uintptr_t)ids & 3) return set_err(ctx, QIMM_ERR_ARG, "qmatmul with adapters: ids must be 4-byte aligned");
    if (m == 0) return QIMM_OK;
    if (const int rc = reserve(ctx, w, ad, m, out_type)) return rc;
    const hipStream_t s = (hipStream_t)stream;
    const Scratch sc = scratch_of(ad, m, out_type);
    float *t = (float *)ctx->ws;
    float *base = out_type == QIMM_TYPE_F32 ? (float *)y : (float *)((char *)ctx->ws + sc.base);
    QIMM_HIP(ctx, qimm::launch_lora_down((const uint16_t *)x_bf16, lda, m, w->cols, ad->table(), (int)ad->count, ids, t,
                                         ad->ldt(), s));
    qimm::EpiParams ep{};
    ep.out = base;
    ep.ldo = w->rows;
    if (qimm::qgemm_workspace(w->gw, m)) {
        ep.part_ws = (float *)ctx->ws_part;
        ep.part_ws_bytes = ctx->ws_part_bytes;
    }
    QIMM_HIP(ctx, qimm::launch_qgemm(w->gw, (const uint16_t *)x_bf16, m, lda, qimm::EPI_F32, ep, s));
    // rows a launch at a time within the grid's limit
    constexpr int64_t MOST = 16 * 65535;
    for (int64_t r = 0; r < m; r += MOST)
        QIMM_HIP(ctx, qimm::launch_lora_up(t + r * ad->ldt(), ad->ldt(), std::min(m - r, MOST), w->rows, ad->table(),
                                           (int)ad->count, ids + r, base + r * w->rows,
                                           out_type == QIMM_TYPE_F32 ? (float *)y + r * w->rows : nullptr,
                                           (uint16_t *)y + r * w->rows, s));
    return QIMM_OK;
}

}  // extern "C"
