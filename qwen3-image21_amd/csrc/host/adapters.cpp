// Low-rank adapters of many requests beside a quantized projection.
#include <string.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "internal.h"

using namespace qimm_host;

struct qimm_adapters {
    qimm_ctx *ctx = nullptr;
    int64_t rows = 0, cols = 0, count = 0, max_rank = 0;
    void *dev = nullptr;  // the table of AdapterDev, then every A and B, then 256 B of zeros
    size_t bytes = 0;
    const qimm::AdapterDev *table() const { return (const qimm::AdapterDev *)dev; }
    const uint16_t *zeros() const { return (const uint16_t *)dev + bytes / 2 - 128; }
    // a part of t, and the k steps of 64 over its parts
    int64_t width() const { return (max_rank + 7) / 8 * 8; }
    int64_t steps(int parts) const { return (parts * width() + 63) / 64; }
};

namespace {

size_t align_up(size_t v) { return (v + 255) & ~(size_t)255; }

// How a product of m rows is taken: each row by itself beside the product's f32 sums (few); or
// t of all rows first, then the rows before the product's tail and the tail, each as k steps of
// the product over bf16 rows (steps) or with a pass over its f32 sums. The pass is for what runs
// over the codes or split over K: its sums are in memory for the reduction anyway, and the pass adds
// them (4096 x 12288 Q4_K at 512 rows 73 us, 84 as steps), while 1024 x 12288 x 4096 takes 106 as
// steps and 121 with it. Only plain outputs have a tail; the others take the pass up to
// PASS_ROWS rows at most where there are bf16 rows, which bounds its sums. Without bf16 rows every
// row has the pass: its sums are held of part_rows rows at a time (PART_SUMS of them, 512 MiB, and
// PART_ROWS rows at most, which fill the card at any width), one part after the other, of one size
// (Q4_K 12288 x 4096 at 16384 rows: all at once 1835 us, 10752 and the rest 1900, two halves 1840).
// Offsets into the scratch: t16 of the steps (or t of the few), t's shares, the f32 sums.
constexpr int64_t PASS_ROWS = 1024;
constexpr int64_t PART_SUMS = (int64_t)1 << 27, PART_ROWS = 16384;
int64_t most_rows(int64_t n) { return std::max<int64_t>(256, std::min(PART_ROWS, PART_SUMS / n / 256 * 256)); }
int64_t part_rows(int64_t n, int64_t rows) {
    const int64_t parts = (rows + most_rows(n) - 1) / most_rows(n);
    return parts <= 1 ? rows : ((rows + parts - 1) / parts + 255) / 256 * 256;
}
struct Route {
    bool few, steps;
    int64_t head, tiles;  // rows before the tail; their tiles of 256
    int64_t part;         // rows of a part of the pass
    int parts;
    size_t shares, sums, total;
};
Route route_of(const qimm_weight *w, const qimm_adapters *ad, int64_t m, int64_t lda, int epi) {
    Route r{};
    const bool plain = epi == qimm::EPI_F32 || epi == qimm::EPI_BF16;
    r.few = qimm::lora_few(m, ad->max_rank, ad->count);
    r.parts = epi == qimm::EPI_F32 ? 3 : 2;
    r.head = m;
    qimm::EpiParams ep{};
    ep.ldo = w->rows;
    ep.part_ws_bytes = qimm::qgemm_workspace(w->gw, m);
    static float some;  // an address: the plans only test for one
    if (ep.part_ws_bytes) ep.part_ws = &some;
    int64_t pass = m;  // rows with a pass
    if (!r.few) {
        if (plain) r.head = m - qimm::qgemm_route(w->gw, m, lda, qimm::EPI_F32, ep).tail;
        const qimm::GemmRoute g = qimm::qgemm_route(w->gw, r.head, lda, qimm::EPI_F32, ep);
        r.steps = g.kernel == qimm::GEMM_BF16_ROWS && g.splits == 1;
        r.tiles = g.head;
        if (!plain && qimm::qgemm_bf16_fits(w->gw) && (r.steps || m > PASS_ROWS)) {
            r.steps = true;
            r.tiles = qimm::qgemm_bf16_plan(w->gw, m, false).head;
        }
        if (r.steps) pass = m - r.head;
        r.shares = r.steps ? align_up((size_t)(m * 64 * ad->steps(r.parts)) * 2) : 0;
        r.sums = r.shares + align_up(qimm::lora_down_scratch(m, w->cols, ad->max_rank));
    } else {
        r.sums = align_up((size_t)(m * ad->max_rank) * 4);
    }
    r.part = epi == qimm::EPI_F32 ? pass : part_rows(w->rows, pass);  // f32 outputs take the sums themselves
    r.total = r.sums + (epi == qimm::EPI_F32 ? 0 : (size_t)(r.part * w->rows) * 4);
    return r;
}

int check_pair(qimm_ctx *ctx, const qimm_weight *w, const qimm_adapters *ad) {
    if (ad->rows != w->rows || ad->cols != w->cols)
        return set_err(ctx, QIMM_ERR_SHAPE, "qmatmul with adapters: the adapters' rows x cols differ from the weight's");
    if (w->ctx->device != ctx->device || ad->ctx->device != ctx->device)
        return set_err(ctx, QIMM_ERR_STATE, "qmatmul with adapters: weight or adapters live on another device");
    return QIMM_OK;
}

int reserve(qimm_ctx *ctx, const qimm_weight *w, int64_t m, const Route &r) {
    if (const int rc = ensure_workspace(ctx, r.total)) return rc;
    const size_t part = adapters_part_workspace(w, m);
    return part ? ensure_part_workspace(ctx, part) : QIMM_OK;
}

int run(qimm_ctx *ctx, const qimm_weight *w, const qimm_adapters *ad, const int32_t *ids, const uint16_t *x, int64_t m,
        int64_t lda, int epi, const qimm::EpiParams &ep, const Route &r, char *ws, hipStream_t s) {
    const int64_t K = w->cols, N = w->rows, steps = ad->steps(r.parts);
    const qimm::AdapterDev *table = ad->table();
    const int n = (int)ad->count;
    float *shares = (float *)(ws + r.shares);
    const qimm::LoraShares sh = qimm::lora_shares(m, K, ad->max_rank);
    if (r.few)
        QIMM_HIP(ctx, qimm::launch_lora_few_down(x, lda, m, K, table, n, ids, shares, ad->max_rank, s));
    else
        QIMM_HIP(ctx, qimm::launch_lora_down(x, lda, m, K, ad->max_rank, table, n, ids, shares, s));
    int64_t row0 = 0;
    if (r.steps) {
        uint16_t *t16 = (uint16_t *)ws;
        QIMM_HIP(ctx, qimm::launch_lora_split(shares, sh, m, ad->width(), r.parts, table, n, ids, t16, 64 * steps, s));
        const qimm::AdapterSteps st{t16, (int)ad->width(), (int)steps, table, n, ids, ad->zeros()};
        QIMM_HIP(ctx, qimm::launch_qgemm_bf16_adapters(w->gw, x, r.head, lda, epi, ep, r.tiles, st, s));
        row0 = r.head;
    }
    if (row0 == m) return QIMM_OK;
    // the rest's f32 sums, to the output where that is f32, and the pass: in parts of whole
    // sequences, or of one that is longer, where the epilogue asks for a row's place in its own
    const int64_t seq = epi == qimm::EPI_QKV ? ep.seq : epi == qimm::EPI_RESID ? ep.g_rows_per : 1;
    for (int64_t at = row0, rows; at < m; at += rows) {
        rows = std::min(seq <= r.part ? r.part / seq * seq : std::min(r.part, seq - at % seq), m - at);
        float *sums = epi == qimm::EPI_F32 ? (float *)ep.out + at * N : (float *)(ws + r.sums);
        float *y32 = epi == qimm::EPI_BF16 ? nullptr : sums;
        uint16_t *y16 = epi == qimm::EPI_BF16 ? (uint16_t *)ep.out + at * N : nullptr;
        qimm::EpiParams es{};
        es.out = sums;
        es.ldo = N;
        es.part_ws = ep.part_ws;
        es.part_ws_bytes = ep.part_ws_bytes;
        qimm::SplitSums base{sums, 1};
        if (!qimm::qgemm_route(w->gw, rows, lda, qimm::EPI_F32, es).tail) es.left = &base;
        QIMM_HIP(ctx, qimm::launch_qgemm(w->gw, x + at * lda, rows, lda, qimm::EPI_F32, es, s));
        if (r.few)
            QIMM_HIP(ctx, qimm::launch_lora_few_up(shares, ad->max_rank, rows, N, table, n, ids, base, y32, y16, s));
        else
            QIMM_HIP(ctx, qimm::launch_lora_up(shares, sh, m, at, rows, N, table, n, ids + at, base, y32, y16, s));
        if (epi != qimm::EPI_F32 && epi != qimm::EPI_BF16)
            QIMM_HIP(ctx, qimm::launch_split_epilogue(sums, 1, rows, N, epi, qimm::rows_from(ep, epi, w->gw, at), s));
    }
    return QIMM_OK;
}

}  // namespace

namespace qimm_host {

int adapters_build(qimm_ctx *ctx, int64_t rows, int64_t cols, const std::vector<HostAdapter> &list, qimm_adapters **out) {
    *out = nullptr;
    const size_t n = list.size();
    std::vector<qimm::AdapterDev> table(n);
    std::vector<size_t> at_a(n), at_b(n);
    size_t off = align_up(n * sizeof(qimm::AdapterDev));
    int64_t max_rank = 0;
    for (size_t i = 0; i < n; i++) {
        const int64_t r = list[i].rank, ldb = (r + 7) / 8 * 8;
        at_a[i] = off;
        off += align_up((size_t)(r * cols) * 2);
        at_b[i] = off;
        off += align_up((size_t)(rows * ldb) * 2);
        max_rank = std::max(max_rank, r);
        for (const std::vector<uint16_t> *v : {&list[i].a, &list[i].b}) {
            bool numbers = true;
            for (const uint16_t x : *v) numbers &= (x & 0x7f80u) != 0x7f80u;
            if (!numbers) return set_err(ctx, QIMM_ERR_ARG, "adapters: values must be numbers within the bf16 range");
        }
    }
    off += 256;  // zeros, which the tiles of other adapters' rows read
    // A as it is; B's rows padded with zeros to 16 bytes
    std::vector<uint8_t> host(off, 0);
    for (size_t i = 0; i < n; i++) {
        const int64_t r = list[i].rank, ldb = (r + 7) / 8 * 8;
        memcpy(&host[at_a[i]], list[i].a.data(), (size_t)(r * cols) * 2);
        for (int64_t row = 0; row < rows; row++)
            memcpy(&host[at_b[i] + (size_t)(row * ldb) * 2], &list[i].b[(size_t)(row * r)], (size_t)r * 2);
    }
    qimm_adapters *ad = new qimm_adapters();
    ad->ctx = ctx;
    ad->rows = rows;
    ad->cols = cols;
    ad->count = (int64_t)n;
    ad->max_rank = max_rank;
    ad->bytes = off;
    hipError_t e = hipSetDevice(ctx->device);
    if (e == hipSuccess) e = hipMalloc(&ad->dev, off);
    if (e == hipSuccess) {
        for (size_t i = 0; i < n; i++) {
            const int r = (int)list[i].rank;
            table[i] = {(const uint16_t *)((char *)ad->dev + at_a[i]), (const uint16_t *)((char *)ad->dev + at_b[i]), r,
                        (r + 7) / 8 * 8, list[i].scale, 0};
        }
        memcpy(host.data(), table.data(), n * sizeof(qimm::AdapterDev));
        e = hipMemcpy(ad->dev, host.data(), off, hipMemcpyHostToDevice);
    }
    if (e != hipSuccess) {
        if (ad->dev) (void)hipFree(ad->dev);
        delete ad;
        return hip_err(ctx, e, "adapters upload");
    }
    *out = ad;
    return QIMM_OK;
}

int adapter_tensors(qimm_ctx *ctx, const qimm_tensor &a, const qimm_tensor &b, int64_t rows, int64_t cols) {
    if (!a.data || !b.data) return set_err(ctx, QIMM_ERR_ARG, "adapters: missing tensor");
    if (a.ggml_type != b.ggml_type ||
        (a.ggml_type != QIMM_TYPE_F32 && a.ggml_type != QIMM_TYPE_F16 && a.ggml_type != QIMM_TYPE_BF16))
        return set_err(ctx, QIMM_ERR_TYPE, "adapters: a and b must both be F32, F16 or BF16");
    const int64_t r = a.rows, e = a.ggml_type == QIMM_TYPE_F32 ? 4 : 2;
    if (r < 1 || r > QIMM_ADAPTER_MAX_RANK || a.cols != cols || b.rows != rows || b.cols != r ||
        a.nbytes != (size_t)(r * cols * e) || b.nbytes != (size_t)(rows * r * e))
        return set_err(ctx, QIMM_ERR_SHAPE, "adapters: a must be [rank, cols] and b [rows, rank], rank 1 to " +
                                                std::to_string(QIMM_ADAPTER_MAX_RANK));
    return QIMM_OK;
}

std::vector<uint16_t> tensor_bf16(const qimm_tensor &t) {
    std::vector<uint16_t> v((size_t)(t.rows * t.cols));
    to_bf16(t.ggml_type, (const uint8_t *)t.data, t.rows * t.cols, v.data());
    return v;
}

size_t adapters_scratch(const qimm_weight *w, const qimm_adapters *ad, int64_t m) {
    const int64_t cus = std::max(qimm::device_cu_count(), 1);
    const qimm::LoraShares one = qimm::lora_shares(m, w->cols, ad->max_rank);
    // t16; the shares, two workgroups of 128 rows per CU or one share; the sums
    const int64_t pass = std::min(most_rows(w->rows), qimm::qgemm_bf16_fits(w->gw) ? std::min(m, PASS_ROWS) : m);
    return align_up((size_t)(m * 64 * ad->steps(2)) * 2) + align_up((size_t)(std::max(m, 2 * cus * 128) * one.ldp) * 4) +
           (size_t)(pass * w->rows) * 4;
}

size_t adapters_part_workspace(const qimm_weight *w, int64_t m) {
    const size_t whole = qimm::qgemm_workspace(w->gw, m);
    // a pass in parts, the last of any size
    const int64_t most = most_rows(w->rows);
    return m <= most ? whole : std::max(whole, qimm::qgemm_workspace_up_to(w->gw, most));
}

int adapted_product(qimm_ctx *ctx, const qimm_weight *w, const qimm_adapters *ad, const int32_t *ids, const uint16_t *x,
                    int64_t m, int64_t lda, int epi, const qimm::EpiParams &ep, char *ws, hipStream_t s) {
    // the hidden state's rounding in a pass of its own, over its f32 values
    const int rounding = epi != qimm::EPI_SWIGLU ? 0 : ep.hmid_q8k ? 256 : ep.hmid_q8_0 ? 32 : 0;
    qimm::EpiParams e = ep;
    e.hmid_q8k = e.hmid_q8_0 = 0;
    const Route r = route_of(w, ad, m, lda, epi);
    if (const int rc = run(ctx, w, ad, ids, x, m, lda, epi, e, r, ws, s)) return rc;
    if (rounding && !ep.hmid_round_later)
        QIMM_HIP(ctx, qimm::launch_quant_rows(ep.hmid_f32, ep.ldh, m, w->rows / 2, rounding, ep.hmid, ep.ldh, s));
    return QIMM_OK;
}

}  // namespace qimm_host

extern "C" {

int qimm_adapters_create(qimm_ctx *ctx, int64_t rows, int64_t cols, const qimm_adapter *list, int64_t n,
                         qimm_adapters **out) {
    if (!ctx || !out || n < 0 || (n > 0 && !list)) return QIMM_ERR_ARG;
    *out = nullptr;
    if (rows <= 0 || rows % 128 || cols <= 0 || cols % 64 || rows >= (int64_t)1 << 31 || cols >= (int64_t)1 << 31)
        return set_err(ctx, QIMM_ERR_SHAPE, "adapters: needs rows % 128 == 0 and cols % 64 == 0");
    if (n < 1 || n > 65535) return set_err(ctx, QIMM_ERR_SHAPE, "adapters: 1 to 65535 of them");
    for (int64_t i = 0; i < n; i++) {
        if (!std::isfinite(list[i].scale)) return set_err(ctx, QIMM_ERR_ARG, "adapters: a scale must be a finite number");
        if (const int rc = adapter_tensors(ctx, list[i].a, list[i].b, rows, cols)) return rc;
    }
    try {
        std::vector<HostAdapter> all((size_t)n);
        for (int64_t i = 0; i < n; i++)
            all[(size_t)i] = {list[i].a.rows, list[i].scale, tensor_bf16(list[i].a), tensor_bf16(list[i].b)};
        return adapters_build(ctx, rows, cols, all, out);
    } catch (const std::bad_alloc &) {
        return set_err(ctx, QIMM_ERR_OOM, "adapters: host staging allocation failed");
    }
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
    const int epi = out_type == QIMM_TYPE_F32 ? qimm::EPI_F32 : qimm::EPI_BF16;
    if (const int rc = reserve(ctx, w, m, route_of(w, ad, m, w->cols, epi))) return rc;
    return reserve(ctx, w, m, route_of(w, ad, m, (int64_t)1 << 40, epi));  // rows too far apart for the bf16 rows' kernel
}

int qimm_qmatmul_adapters(qimm_ctx *ctx, const qimm_weight *w, const qimm_adapters *ad, const int32_t *ids,
                          const void *x_bf16, int64_t m, int64_t lda, void *y, int out_type, void *stream) {
    if (!ad || !ids) return QIMM_ERR_ARG;
    if (const int rc = qmatmul_check(ctx, w, x_bf16, m, lda, y, out_type)) return rc;
    if (const int rc = check_pair(ctx, w, ad)) return rc;
    if ((uintptr_t)ids & 3) return set_err(ctx, QIMM_ERR_ARG, "qmatmul with adapters: ids must be 4-byte aligned");
    if (m == 0) return QIMM_OK;
    QIMM_HIP(ctx, hipSetDevice(ctx->device));
    const int epi = out_type == QIMM_TYPE_F32 ? qimm::EPI_F32 : qimm::EPI_BF16;
    const Route r = route_of(w, ad, m, lda, epi);
    if (const int rc = reserve(ctx, w, m, r)) return rc;
    qimm::EpiParams ep{};
    ep.out = y;
    ep.ldo = w->rows;
    if (adapters_part_workspace(w, m)) {
        ep.part_ws = (float *)ctx->ws_part;
        ep.part_ws_bytes = ctx->ws_part_bytes;
    }
    return run(ctx, w, ad, ids, (const uint16_t *)x_bf16, m, lda, epi, ep, r, (char *)ctx->ws, (hipStream_t)stream);
}

}  // extern "C"
