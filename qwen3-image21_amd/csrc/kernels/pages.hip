// Page tables of a step built on the device, and the store of rows into pages and back, gfx950.
//
// The plan. Request r has old_r tokens and adds a_r; with the sums over the requests before it,
// start_r of rows and base_r of new pages, its page k from ceil(old_r / ps) on is entry base_r + ... of
// the queue of free pages, and the slot of a token at position p is table[p / ps] ps + p % ps. Bound by
// latency: a few bytes a request and 8 a row. One workgroup makes the sums in registers and LDS.
//
// The store. Bound by bytes: a key's 8 dims are 16 B of its granule, four keys' values of one dim 8 B
// (paged.h), so a thread takes 8 dims of four rows and turns their values over in registers where
// the four rows are four consecutive slots; rows that are not (the ends of a request) write
// their values one by one.
#include <type_traits>

#include "device_common.h"
#include "paged.h"

namespace qimm {
namespace {

constexpr int PLAN_THREADS = 1024;

// exclusive sums of v over the workgroup's threads, and the total; `part` takes a value per wave
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t *part, int64_t &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t x = __shfl_up(s, o);
        if (lane >= o) s += x;
    }
    __syncthreads();  // part may still be read by an earlier call
    if (lane == 63) part[wave] = s;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int w = 0; w < (int)(blockDim.x >> 6); w++) {
        if (w < wave) before += part[w];
        total += part[w];
    }
    return before + s - v;
}

// A request's step. fits: it adds tokens, and its table and the rows have room for them.
struct Step {
    int old, add, have;  // tokens, tokens added (negative: given back), pages held
    int64_t end;         // rows up to and with it
    bool fits;
    int need;            // new pages, 0 where it does not fit
    int freed;           // pages given back
};

__device__ __forceinline__ Step step_of(const PagePlanArgs &p, int64_t r, int64_t rows_before) {
    Step s;
    s.old = p.lengths[r];
    s.add = p.added[r];
    const int ps = p.page_size;
    const int64_t room = p.max_pages * ps, after = (int64_t)s.old + s.add;
    s.have = s.old > 0 ? (int)min(((int64_t)s.old + ps - 1) / ps, p.max_pages) : 0;
    s.end = rows_before + max(s.add, 0);
    s.fits = s.add > 0 && s.old >= 0 && after <= room && s.end <= p.max_rows;
    s.need = s.fits ? (int)((after + ps - 1) / ps) - s.have : 0;
    s.freed = s.add < 0 ? s.have : 0;
    return s;
}

// entry i of the queue after its head, i < 2 * pages
__device__ __forceinline__ int32_t *queue_at(const PagePlanArgs &p, int head, int64_t i) {
    int64_t at = head + i;
    while (at >= p.pages) at -= p.pages;
    return p.queue + at;
}

// Row t's slot and position, and the table entry of a page that starts with it. start, old, base
// (queue entries before the request's first new page, -1: not served) are its request's.
__device__ __forceinline__ void fill_row(const PagePlanArgs &p, int64_t t, int64_t r, int start, int old, int base, int head) {
    int slot = -1, pos = 0;
    if (base >= 0) {
        pos = old + (int)(t - start);
        const int ps = p.page_size, k = pos / ps, in = pos - k * ps, have = (int)(((int64_t)old + ps - 1) / ps);
        int32_t *entry = p.tables + r * p.max_pages + k;
        const int page = k < have ? *entry : *queue_at(p, head, (int64_t)base + k - have);
        if (k >= have && in == 0) *entry = page;
        if (page >= 0 && page < p.pages) slot = page * ps + in;
    }
    p.slots[t] = slot;
    if (p.positions) p.positions[t] = pos;
}

// The sums of a step by one workgroup: starts, lengths_out, state_out, and per request in work
// {start, old, base, entries before its first page given back (-1: none)}, then {head, free}.
__global__ __launch_bounds__(PLAN_THREADS) void page_plan_kernel(const PagePlanArgs p) {
    __shared__ int64_t part[PLAN_THREADS / 64];
    const int tid = threadIdx.x;
    const int64_t R = p.requests, c = (R + PLAN_THREADS - 1) / PLAN_THREADS;
    const int64_t r0 = min(tid * c, R), r1 = min(r0 + c, R);
    const int free = (int)min((int64_t)max(p.state[1], 0), p.pages);
    int head = (int)(p.state[0] % p.pages);
    if (head < 0) head += (int)p.pages;

    int64_t rows = 0, rows_all, need = 0, need_all, freed = 0, freed_all;
    for (int64_t r = r0; r < r1; r++) rows += max(p.added[r], 0);
    const int64_t rows0 = block_scan(rows, part, rows_all);
    int64_t end = rows0;
    for (int64_t r = r0; r < r1; r++) {
        const Step s = step_of(p, r, end);
        end = s.end;
        need += s.need;
        freed += s.freed;
    }
    int64_t cum = block_scan(need, part, need_all);
    int64_t back = block_scan(freed, part, freed_all);
    int64_t taken = 0, refused = 0;
    end = rows0;
    for (int64_t r = r0; r < r1; r++) {
        const Step s = step_of(p, r, end);
        const bool served = s.fits && (s.need == 0 || cum + s.need <= free);
        const int start = (int)min(end, p.max_rows);
        p.starts[r] = start;
        int32_t *w = p.work + 4 * r;
        w[0] = start;
        w[1] = s.old;
        w[2] = served ? (s.need ? (int)cum : 0) : -1;
        w[3] = s.freed ? (int)min(back, (int64_t)0x7fffffff) : -1;
        p.lengths_out[r] = s.add < 0 ? 0 : served ? s.old + s.add : s.old;
        taken += served ? s.need : 0;
        refused += s.add > 0 && !served;
        end = s.end;
        cum += s.need;
        back += s.freed;
    }
    int64_t taken_all, refused_all;
    block_scan(taken, part, taken_all);
    block_scan(refused, part, refused_all);
    const int all = (int)min(rows_all, p.max_rows);
    if (tid == 0) {
        p.starts[R] = all;
        int64_t at = head + taken_all;
        if (at >= p.pages) at -= p.pages;
        p.state_out[0] = (int)at;
        p.state_out[1] = (int)min(free - taken_all + freed_all, p.pages);
        p.state_out[2] = all;
        p.state_out[3] = (int)refused_all;
        p.work[4 * R] = head;
        p.work[4 * R + 1] = free;
    }
}

// Slots, positions and table entries of the rows, then the queue entries of the pages given back.
__global__ __launch_bounds__(256) void page_fill_kernel(const PagePlanArgs p) {
    const int64_t R = p.requests;
    const int head = p.work[4 * R], free = p.work[4 * R + 1], all = p.starts[R];
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t < all) {
        int64_t lo = 0, hi = R;  // starts[lo] <= t < starts[hi]
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (p.starts[mid] <= t)
                lo = mid;
            else
                hi = mid;
        }
        const int32_t *w = p.work + 4 * lo;
        fill_row(p, t, lo, w[0], w[1], w[2], head);
    } else if (t < p.max_rows) {
        p.slots[t] = -1;
        if (p.positions) p.positions[t] = 0;
    }
    const int lane = threadIdx.x & 63;
    const int64_t waves = (int64_t)gridDim.x * 4;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < R; r += waves) {
        const int back = p.work[4 * r + 3];
        if (back < 0) continue;
        const int have = (int)min(((int64_t)p.work[4 * r + 1] + p.page_size - 1) / p.page_size, p.max_pages);
        // (entries past the queue's size would be pages given back twice)
        for (int k = lane; k < have && (int64_t)free + back + k < 2 * p.pages; k += 64)
            *queue_at(p, head, (int64_t)free + back + k) = p.tables[r * p.max_pages + k];
    }
}

// ---- rows to slots and back ----

template <typename T>
__device__ __forceinline__ u32x4 load8_bf16(const T *p);
template <>
__device__ __forceinline__ u32x4 load8_bf16<__bf16>(const __bf16 *p) {
    return *(const u32x4 *)p;
}
template <>
__device__ __forceinline__ u32x4 load8_bf16<float>(const float *p) {
    const f32x4 a = ((const f32x4 *)p)[0], b = ((const f32x4 *)p)[1];
    return u32x4{pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3])};
}
template <>
__device__ __forceinline__ u32x4 load8_bf16<_Float16>(const _Float16 *p) {
    const u32x4 w = *(const u32x4 *)p;
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = pack_bf16x2(f16_to_f32(w[i]), f16_to_f32(w[i] >> 16));
    return o;
}

// dim e (0 .. 7) of four rows' 8 dims, in row order
__device__ __forceinline__ u32x2 column(const u32x4 (&x)[4], int e) {
    const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;  // the high / low halves of two words
    return u32x2{__builtin_amdgcn_perm(x[1][e >> 1], x[0][e >> 1], sel), __builtin_amdgcn_perm(x[3][e >> 1], x[2][e >> 1], sel)};
}

// T: the rows' type; STORE: into the pages, else out of them (bf16)
template <typename T, bool STORE, int D>
__global__ __launch_bounds__(256) void pages_rows_kernel(PageDims d, uint8_t *layer, T *k, T *v, int64_t k_row, int64_t k_head,
                                                         int64_t v_row, int64_t v_head, const int32_t *__restrict__ slots,
                                                         int64_t rows) {
    constexpr int OCT = D / 8, GROUPS = 256 / OCT;
    const int o = threadIdx.x % OCT, h = blockIdx.y;
    const int64_t t0 = ((int64_t)blockIdx.x * GROUPS + threadIdx.x / OCT) * 4;
    if (t0 >= rows) return;
    const int64_t most = d.pages * d.page_size;
    // the slots of rows t0 - 3 .. t0 + 6
    int s[10];
#pragma unroll
    for (int i = 0; i < 10; i++) {
        const int64_t t = t0 + i - 3;
        const int x = t >= 0 && t < rows ? slots[t] : -1;
        s[i] = x >= 0 && x < most ? x : -1;
    }
    auto granule = [&](int slot) __attribute__((always_inline)) {
        const int page = slot / d.page_size, in = slot - page * d.page_size;
        return layer + (((int64_t)page * d.kv_heads + h) * (d.page_size >> 4) + (in >> 4)) * granule_bytes(D);
    };
    // whether row t0 + j (j = -3 .. 3) leads four rows with the four slots of a quad
    auto leads = [&](int j) __attribute__((always_inline)) {
        const int x = s[j + 3];
        return x >= 0 && (x & 3) == 0 && s[j + 4] == x + 1 && s[j + 5] == x + 2 && s[j + 6] == x + 3;
    };
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int64_t t = t0 + j;
        const int x = s[j + 3];
        if (t >= rows) break;
        T *kp = k + t * k_row + h * k_head + o * 8;
        if (x < 0) {
            if constexpr (!STORE) {
                *(u32x4 *)kp = u32x4{};
                *(u32x4 *)(v + t * v_row + h * v_head + o * 8) = u32x4{};
            }
            continue;
        }
        uint8_t *g = granule(x);
        u32x4 *kc = (u32x4 *)(g + granule_k(x & 15, o * 8));
        if constexpr (STORE)
            *kc = load8_bf16(kp);
        else
            *(u32x4 *)kp = *kc;
        if (leads(j)) {
            u32x4 y[4];
            if constexpr (STORE) {
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = load8_bf16(v + (t + i) * v_row + h * v_head + o * 8);
#pragma unroll
                for (int e = 0; e < 8; e++) *(u32x2 *)(g + granule_v(D, x & 15, o * 8 + e)) = column(y, e);
            } else {
                u32x2 c[8];
#pragma unroll
                for (int e = 0; e < 8; e++) c[e] = *(const u32x2 *)(g + granule_v(D, x & 15, o * 8 + e));
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t sel = i & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
                    for (int w = 0; w < 4; w++) y[i][w] = __builtin_amdgcn_perm(c[2 * w + 1][i >> 1], c[2 * w][i >> 1], sel);
                    *(u32x4 *)(v + (t + i) * v_row + h * v_head + o * 8) = y[i];
                }
            }
            continue;
        }
        // rows t - (x & 3) .. of one quad are their leader's
        bool led = false;
#pragma unroll
        for (int i = 1; i < 4; i++) led = led || ((x & 3) == i && leads(j - i));
        if (led) continue;
        u32x4 y;
        T *vp = v + t * v_row + h * v_head + o * 8;
        if constexpr (STORE) y = load8_bf16(vp);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            uint16_t *c = (uint16_t *)(g + granule_v(D, x & 15, o * 8 + e));
            if constexpr (STORE)
                *c = (uint16_t)(y[e >> 1] >> (16 * (e & 1)));
            else
                y[e >> 1] = e & 1 ? y[e >> 1] | (uint32_t)*c << 16 : (uint32_t)*c;
        }
        if constexpr (!STORE) *(u32x4 *)vp = y;
    }
}

template <typename T, bool STORE>
hipError_t launch_rows(const PageDims &d, uint8_t *layer, T *k, T *v, int64_t k_row, int64_t k_head, int64_t v_row,
                       int64_t v_head, const int32_t *slots, int64_t rows, hipStream_t stream) {
    if (rows <= 0) return hipSuccess;
    const int per = 256 / (d.head_dim / 8) * 4;
    const int64_t blocks = (rows + per - 1) / per;
    if (blocks >= (int64_t)1 << 24 || d.kv_heads > 65535) return hipErrorInvalidValue;
    const dim3 grid((unsigned)blocks, (unsigned)d.kv_heads);
    if (d.head_dim == 128)
        pages_rows_kernel<T, STORE, 128><<<grid, 256, 0, stream>>>(d, layer, k, v, k_row, k_head, v_row, v_head, slots, rows);
    else if (d.head_dim == 64)
        pages_rows_kernel<T, STORE, 64><<<grid, 256, 0, stream>>>(d, layer, k, v, k_row, k_head, v_row, v_head, slots, rows);
    else
        return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace

hipError_t launch_page_plan(const PagePlanArgs &p, hipStream_t stream) {
    const int64_t blocks = (p.max_rows + 255) / 256;
    if (p.requests <= 0 || p.pages <= 0 || blocks >= (int64_t)1 << 24) return hipErrorInvalidValue;
    page_plan_kernel<<<1, PLAN_THREADS, 0, stream>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    page_fill_kernel<<<(unsigned)(blocks > 0 ? blocks : 1), 256, 0, stream>>>(p);
    return hipGetLastError();
}

hipError_t launch_pages_store(const PageDims &d, uint8_t *layer, const void *k, const void *v, int type, int64_t k_row,
                              int64_t k_head, int64_t v_row, int64_t v_head, const int32_t *slots, int64_t rows,
                              hipStream_t stream) {
    switch (type) {
    case 0: return launch_rows<float, true>(d, layer, (float *)k, (float *)v, k_row, k_head, v_row, v_head, slots, rows, stream);
    case 1: return launch_rows<_Float16, true>(d, layer, (_Float16 *)k, (_Float16 *)v, k_row, k_head, v_row, v_head, slots, rows, stream);
    case 30: return launch_rows<__bf16, true>(d, layer, (__bf16 *)k, (__bf16 *)v, k_row, k_head, v_row, v_head, slots, rows, stream);
    default: return hipErrorInvalidValue;
    }
}

hipError_t launch_pages_load(const PageDims &d, const uint8_t *layer, uint16_t *k, uint16_t *v, const int32_t *slots,
                             int64_t rows, hipStream_t stream) {
    const int64_t row = (int64_t)d.kv_heads * d.head_dim;
    return launch_rows<__bf16, false>(d, const_cast<uint8_t *>(layer), (__bf16 *)k, (__bf16 *)v, row, d.head_dim, row,
                                      d.head_dim, slots, rows, stream);
}

}  // namespace qimm
