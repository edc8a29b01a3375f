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
    const uint16_t *zeros() const { return (const uint16_t *)dev + bytes / 2 - 128; }  // the last 256 B
};

namespace {

size_t align_up(size_t v) { return (v + 255) & ~(size_t)255; }

// How a product of m rows is taken: each row by itself beside the product's f32 sums (few); or
// t of all rows first, then the rows before the product's tail and the tail, each as k steps of
// the product over bf16 rows (steps) or with a pass over its f32 sums. The pass is for what runs
// over the codes or split over K: its sums are in memory for the reduction anyway (4096 x 12288
// Q4_K at 128 / 512 rows 51 / 79 us, 63 / 84 as steps), while 1024 x 12288 x 4096 takes 106 as
// steps and 121 with it. Offsets into the context's growable workspace: t16 of the steps,
// t's shares, the f32 sums of a bf16 output; `part`: the split products' own scratch.
struct Route {
    bool few, steps;
    int64_t head, tiles;  // rows before the tail; their tiles of 256
    int parts;
    size_t shares, sums, total, part;
};
Route route_of(const qimm_weight *w, const qimm_adapters *ad, int64_t m, int64_t lda, int out_type) {
    Route r{};
    const bool f32 = out_type == QIMM_TYPE_F32;
    const int64_t kt = (ad->max_rank + 63) / 64 * 64;
    r.few = qimm::lora_few(m);
    r.parts = f32 ? 3 : 2;
    r.head = m;
    r.part = qimm::qgemm_workspace(w->gw, m);
    qimm::EpiParams ep{};
    ep.ldo = w->rows;
    ep.part_ws_bytes = r.part;
    static float some;  // an address: the plans only test for one
    if (r.part) ep.part_ws = &some;
    int64_t pass = m;  // rows with a pass
    if (!r.few) {
        r.head = m - qimm::qgemm_route(w->gw, m, lda, qimm::EPI_F32, ep).tail;
        const qimm::GemmRoute g = qimm::qgemm_route(w->gw, r.head, lda, qimm::EPI_F32, ep);
        r.steps = g.kernel == qimm::GEMM_BF16_ROWS && g.splits == 1;
        r.tiles = g.head;
        if (r.steps) pass = m - r.head;
        r.shares = r.steps ? align_up((size_t)(m * r.parts * kt) * 2) : 0;
        r.sums = r.shares + align_up(qimm::lora_down_scratch(m, w->cols, ad->max_rank));
    } else {
        r.sums = align_up((size_t)(m * ad->max_rank) * 4);
    }
    r.total = r.sums + (f32 ? 0 : (size_t)(pass * w->rows) * 4);
    return r;
}

int check_pair(qimm_ctx *ctx, const qimm_weight *w, const qimm_adapters *ad) {
    if (ad->rows != w->rows || ad->cols != w->cols)
        return set_err(ctx, QIMM_ERR_SHAPE, "qmatmul with adapters: the adapters' rows x cols differ from the weight's");
    if (w->ctx->device != ctx->device || ad->ctx->device != ctx->device)
        return set_err(ctx, QIMM_ERR_STATE, "qmatmul with adapters: weight or adapters live on another device");
    return QIMM_OK;
}

int reserve(qimm_ctx *ctx, const Route &r) {
    if (const int rc = ensure_workspace(ctx, r.total)) return rc;
    return r.part ? ensure_part_workspace(ctx, r.part) : QIMM_OK;
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
        off += 256;  // zeros, which the tiles of other adapters' rows read
        ad->bytes = off;
        // A as it is; B's rows padded with zeros to 16 bytes
        std::vector<uint8_t> host(off, 0);
        for (int64_t i = 0; i < n; i++) {
            const int64_t r = list[i].a.rows, ldb = (r + 7) / 8 * 8;
            to_bf16(list[i].a.ggml_type, (const uint8_t *)list[i].a.data, r * cols, (uint16_t *)&host[at_a[(size_t)i]]);
            std::vector<uint16_t> b((size_t)(rows * r));
            to_bf16(list[i].b.ggml_type, (const uint8_t *)list[i].b.data, rows * r, b.data());
            for (const uint16_t *p : {(const uint16_t *)&host[at_a[(size_t)i]], (const uint16_t *)b.data()}) {
                const int64_t count = p == b.data() ? rows * r : r * cols;
                bool numbers = true;
                for (int64_t q = 0; q < count; q++) numbers &= (p[q] & 0x7f80u) != 0x7f80u;
                if (!numbers) {
                    delete ad;
                    return set_err(ctx, QIMM_ERR_ARG, "adapters: values must be numbers within the bf16 range");
                }
            }
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
    if (m == 0) return QIMM_OK;
    QIMM_HIP(ctx, hipSetDevice(ctx->device));
    if (const int rc = reserve(ctx, route_of(w, ad, m, w->cols, out_type))) return rc;
    return reserve(ctx, route_of(w, ad, m, (int64_t)1 << 40, out_type));  // rows too far apart for the bf16 rows' kernel
}

int qimm_qmatmul_adapters(qimm_ctx *ctx, const qimm_weight *w, const qimm_adapters *ad, const int32_t *ids,
                          const void *x_bf16, int64_t m, int64_t lda, void *y, int out_type, void *stream) {
    if (!ad || !ids) return QIMM_ERR_ARG;
    if (const int rc = qmatmul_check(ctx, w, x_bf16, m, lda, y, out_type)) return rc;
    if (const int rc = check_pair(ctx, w, ad)) return rc;
    if ((uintptr_t)ids & 3) return set_err(ctx, QIMM_ERR_ARG, "qmatmul with adapters: ids must be 4-byte aligned");
    if (m == 0) return QIMM_OK;
    QIMM_HIP(ctx, hipSetDevice(ctx->device));
    const Route r = route_of(w, ad, m, lda, out_type);
    if (const int rc = reserve(ctx, r)) return rc;
    const hipStream_t s = (hipStream_t)stream;
    const uint16_t *x = (const uint16_t *)x_bf16;
    const bool f32 = out_type == QIMM_TYPE_F32;
    const int64_t K = w->cols, N = w->rows, kt = (ad->max_rank + 63) / 64 * 64;
    const qimm::AdapterDev *table = ad->table();
    const int n = (int)ad->count;
    char *ws = (char *)ctx->ws;
    uint16_t *t16 = (uint16_t *)ws;
    float *shares = (float *)(ws + r.shares);
    const qimm::LoraShares sh = qimm::lora_shares(m, K, ad->max_rank);
    qimm::EpiParams ep{};
    ep.ldo = N;
    if (r.part) {
        ep.part_ws = (float *)ctx->ws_part;
        ep.part_ws_bytes = ctx->ws_part_bytes;
    }
    if (r.few)
        QIMM_HIP(ctx, qimm::launch_lora_few_down(x, lda, m, K, table, n, ids, shares, ad->max_rank, s));
    else
        QIMM_HIP(ctx, qimm::launch_lora_down(x, lda, m, K, ad->max_rank, table, n, ids, shares, s));
    int64_t row0 = 0;
    if (r.steps) {
        QIMM_HIP(ctx, qimm::launch_lora_split(shares, sh, m, kt, r.parts, table, n, ids, t16, s));
        const qimm::AdapterSteps st{t16, (int)(kt / 64), (int)(kt / 64) * r.parts, table, n, ids, ad->zeros()};
        ep.out = y;
        QIMM_HIP(ctx, qimm::launch_qgemm_bf16_adapters(w->gw, x, r.head, lda, f32 ? qimm::EPI_F32 : qimm::EPI_BF16, ep, r.tiles, st, s));
        row0 = r.head;
    }
    if (row0 == m) return QIMM_OK;
    float *y32 = f32 ? (float *)y + row0 * N : nullptr, *sums = f32 ? y32 : (float *)(ws + r.sums);
    uint16_t *y16 = (uint16_t *)y + row0 * N;
    ep.out = sums;
    QIMM_HIP(ctx, qimm::launch_qgemm(w->gw, x + row0 * lda, m - row0, lda, qimm::EPI_F32, ep, s));
    if (r.few)
        QIMM_HIP(ctx, qimm::launch_lora_few_up(shares, ad->max_rank, m, N, table, n, ids, sums, y32, y16, s));
    else
        QIMM_HIP(ctx, qimm::launch_lora_up(shares, sh, m, row0, m - row0, N, table, n, ids + row0, sums, y32, y16, s));
    return QIMM_OK;
}

}  // extern "C"
