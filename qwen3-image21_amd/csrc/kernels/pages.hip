// Page tables of a step built on the device, and the store of rows into pages and back, gfx950.
//
// The plan. Request r has old_r tokens and adds a_r; with the sums over the requests before it,
// start_r of rows and base_r of new pages, its page k from ceil(old_r / ps) on is entry base_r + ... of
// the queue of free pages, and the slot of a token at position p is table[p / ps] ps + p % ps. Bound by
// latency: a few bytes a request and 8 a row, so reads that do not depend on each other are made together. One workgroup
// makes the sums in registers; where requests and rows are few it writes the rows too, from LDS, else a second
// launch does. 48 requests of a token: 3.0 us; 2048 requests, 128 of them of 509 tokens: 5.3 and 6.7.
//
// The store. Bound by bytes. Where 16 rows are the 16 slots of a granule, in order, a wave takes them: keys as
// they are read are written 1 KB in a row, values are turned over in registers, four rows and eight dims a
// lane, and gathered in LDS (paged.h). Other rows, the ends of a request and single tokens, are
// written 16 B of a key and 2 B of a value at a time. 8395 rows of 32 heads of 128: f32 88 us (4.7 TB/s), bf16
// 55 to 60, f16 59 to 65, back 51.
#include <algorithm>
#include <type_traits>

#include "device_common.h"
#include "paged.h"

namespace qimm {
namespace {

constexpr int PLAN_REQUESTS = 1024, PLAN_ROWS = 2048;  // what one launch takes

// four int32 of the plan's work, which is aligned as its caller's int32 are
typedef int work4 __attribute__((ext_vector_type(4), aligned(4)));

// A step's sums over the requests, in 32 bits that stop at the largest number: rows up to max_rows, pages up
// to those that are free and back to the queue are all that counts.
struct Sums {
    uint32_t rows, need, freed;
};
__device__ __forceinline__ Sums add(Sums a, Sums b) {
    return {__builtin_elementwise_add_sat(a.rows, b.rows), __builtin_elementwise_add_sat(a.need, b.need),
            __builtin_elementwise_add_sat(a.freed, b.freed)};
}
template <int CTRL, int ROWS>
__device__ __forceinline__ Sums scan_step(Sums s) {
    const auto from = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false); };
    return add(s, {from(s.rows), from(s.need), from(s.freed)});
}
// those of the threads before this one, and of all; `part` takes a value per wave
template <int THREADS>
__device__ __forceinline__ Sums block_scan(Sums v, Sums *part, Sums &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Sums s = v;
    s = scan_step<0x111, 0xf>(s);  // row_shr 1, 2, 4, 8
    s = scan_step<0x112, 0xf>(s);
    s = scan_step<0x114, 0xf>(s);
    s = scan_step<0x118, 0xf>(s);
    s = scan_step<0x142, 0xa>(s);  // row_bcast 15, 31
    s = scan_step<0x143, 0xc>(s);
    if (lane == 63) part[wave] = s;
    __syncthreads();
    Sums before{0, 0, 0};
    total = before;
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) {
        if (w == wave) before = total;
        total = add(total, part[w]);
    }
    const Sums up{(uint32_t)__shfl_up((int)s.rows, 1), (uint32_t)__shfl_up((int)s.need, 1), (uint32_t)__shfl_up((int)s.freed, 1)};
    return lane ? add(before, up) : before;
}

// A request's step. fits: it adds tokens and its table has room for them.
struct Step {
    int old, add, have;  // tokens, tokens added (negative: given back), pages held
    bool fits;
    int need;            // new pages, 0 where it does not fit
    int freed;           // pages given back
    __device__ Sums sums() const { return {(uint32_t)max(add, 0), (uint32_t)need, (uint32_t)freed}; }
};

__device__ __forceinline__ Step step_of(const PagePlanArgs &p, int64_t r) {
    Step s;
    s.old = p.lengths[r];
    s.add = p.added[r];
    const int ps = p.page_size;
    // (lengths and positions are 32 bits, a table may be wider)
    const int64_t room = min(p.max_pages * ps, (int64_t)0x7fffffff), after = (int64_t)s.old + s.add;
    s.have = s.old > 0 ? (int)min(((int64_t)s.old + ps - 1) / ps, p.max_pages) : 0;
    s.fits = s.add > 0 && s.old >= 0 && after <= room;
    s.need = s.fits ? (int)((after + ps - 1) / ps) - s.have : 0;
    s.freed = s.add < 0 ? s.have : 0;
    return s;
}

// entry i of the queue after its head, i < pages
__device__ __forceinline__ int32_t *queue_at(const PagePlanArgs &p, int head, int64_t i) {
    int64_t at = head + i;
    if (at >= p.pages) at -= p.pages;
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

// The pages of a request given back, `lane` of 64: `back` entries of the queue come before its first.
__device__ __forceinline__ void give_back(const PagePlanArgs &p, int64_t r, int old, int64_t back, int head, int free, int lane) {
    const int have = (int)min(((int64_t)old + p.page_size - 1) / p.page_size, p.max_pages);
    // (more pages than the queue has room for are pages given back twice: those that are free stay)
    for (int k = lane; k < have && free + back + k < p.pages; k += 64)
        *queue_at(p, head, free + back + k) = p.tables[r * p.max_pages + k];
}

// The pages of all requests given back, wave `wave` of `waves`: of its requests, every `waves`-th, a lane each
// looks whether it is one. of(r): {, old, , entries before its first page (-1: not given back)}.
template <typename OF>
__device__ __forceinline__ void give_back_all(const PagePlanArgs &p, int64_t wave, int64_t waves, int head, int free, OF of) {
    const int lane = threadIdx.x & 63;
    for (int64_t r0 = wave; r0 < p.requests; r0 += 64 * waves) {
        const int64_t r = r0 + lane * waves;
        const int4 w = r < p.requests ? of(r) : make_int4(0, 0, 0, -1);
        for (uint64_t some = __ballot(w.w >= 0); some; some &= some - 1) {
            const int i = __builtin_ctzll(some);
            give_back(p, r0 + i * waves, __builtin_amdgcn_readlane(w.y, i), __builtin_amdgcn_readlane(w.w, i), head, free, lane);
        }
    }
}

// The sums of a step by one workgroup: starts, lengths_out, state_out, and of every request {start, old,
// base, entries before its first page given back (-1: none)}: in LDS (FILL: up to PLAN_REQUESTS), for
// the rows, which it then writes; or in work, then {head, free}. A request that fits within the rows has
// only such before it, so the sums need not ask for it.
// HELD: the requests of a thread, in registers (their lengths are read together, which took the launch for 2048
// requests from 6.3 to 5.3 us); 0: any number, read twice.
template <int THREADS, bool FILL, int HELD>
__global__ __launch_bounds__(THREADS) void page_plan_kernel(const PagePlanArgs p) {
    __shared__ Sums part[THREADS / 64];
    __shared__ int taken, refused;
    __shared__ int4 of[FILL ? THREADS : 1];
    __shared__ int starts[FILL ? THREADS + 1 : 1];
    const int tid = threadIdx.x;
    const int64_t R = p.requests, c = FILL ? 1 : (R + THREADS - 1) / THREADS;
    const int64_t r0 = min(tid * c, R), r1 = min(r0 + c, R);
    if (tid == 0) taken = refused = 0;
    const int free = (int)min((int64_t)max(p.state[1], 0), p.pages);
    int head = (int)(p.state[0] % p.pages);
    if (head < 0) head += (int)p.pages;

    Sums mine{0, 0, 0}, all;
    Step held[HELD ? HELD : 1];
    if constexpr (HELD > 0) {
#pragma unroll
        for (int i = 0; i < HELD; i++)
            if (r0 + i < r1) held[i] = step_of(p, r0 + i);
#pragma unroll
        for (int i = 0; i < HELD; i++)
            if (r0 + i < r1) mine = add(mine, held[i].sums());
    } else {
        for (int64_t r = r0; r < r1; r++) mine = add(mine, step_of(p, r).sums());
    }
    Sums at = block_scan<THREADS>(mine, part, all);
    const uint32_t most = (uint32_t)p.max_rows;
    int used = 0, no = 0;
    auto settle = [&](int64_t r, const Step &s) __attribute__((always_inline)) {
        const Sums end = add(at, s.sums());
        const bool served = s.fits && end.rows <= most && (s.need == 0 || end.need <= (uint32_t)free);
        const int start = (int)min(at.rows, most);
        const int4 w = make_int4(start, s.old, served ? (s.need ? (int)at.need : 0) : -1, s.freed ? (int)min(at.freed, 0x7fffffffu) : -1);
        if (FILL) {
            of[tid] = w;
            starts[tid] = start;
        } else {
            *(work4 *)(p.work + 4 * r) = work4{w.x, w.y, w.z, w.w};
        }
        p.starts[r] = start;
        p.lengths_out[r] = s.add < 0 ? 0 : served ? s.old + s.add : s.old;
        if (served && s.need) used = (int)end.need;
        no += s.add > 0 && !served;
        at = end;
    };
    if constexpr (HELD > 0) {
#pragma unroll
        for (int i = 0; i < HELD; i++)
            if (r0 + i < r1) settle(r0 + i, held[i]);
    } else {
        for (int64_t r = r0; r < r1; r++) settle(r, step_of(p, r));
    }
    if (used) atomicMax(&taken, used);
    if (no) atomicAdd(&refused, no);
    __syncthreads();
    const int rows = (int)min(all.rows, most);
    if (tid == 0) {
        p.starts[R] = rows;
        int64_t to = (int64_t)head + taken;
        if (to >= p.pages) to -= p.pages;
        p.state_out[0] = (int)to;
        p.state_out[1] = free - taken + (int)min((int64_t)all.freed, p.pages - free);
        p.state_out[2] = rows;
        p.state_out[3] = refused;
        if (!FILL) {
            p.work[4 * R] = head;
            p.work[4 * R + 1] = free;
        }
    }
    if constexpr (FILL) {
        for (int64_t t = tid; t < p.max_rows; t += THREADS) {
            if (t >= rows) {
                p.slots[t] = -1;
                if (p.positions) p.positions[t] = 0;
                continue;
            }
            int lo = 0, hi = (int)R;  // starts[lo] <= t < starts[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (starts[mid] <= t)
                    lo = mid;
                else
                    hi = mid;
            }
            const int4 w = of[lo];
            fill_row(p, t, lo, w.x, w.y, w.z, head);
        }
        if (all.freed)
            give_back_all(p, tid >> 6, THREADS / 64, head, free, [&](int64_t r) { return of[r]; });
    }
}

// The largest of `n` requests whose rows start at or before t (starts[0] is 0), by a wave: 64 at a time.
__device__ __forceinline__ int64_t request_of(const int32_t *starts, int64_t n, int64_t t) {
    const int lane = threadIdx.x & 63;
    int64_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const int64_t step = (hi - lo + 63) / 64, at = lo + lane * step;
        const int k = __popcll(__ballot(at < hi && starts[min(at, hi - 1)] <= t));
        lo += max(k - 1, 0) * step;
        hi = min(lo + step, hi);
    }
    return lo;
}

// Slots, positions and table entries of the rows, then the queue entries of the pages given back. Starts of up to
// HELD requests are all read into LDS, of more those of the workgroup's rows. Workgroups behind the rows only give
// pages back.
__global__ __launch_bounds__(256) void page_fill_kernel(const PagePlanArgs p) {
    constexpr int HELD = 4096;
    __shared__ int starts[HELD];
    __shared__ int64_t ends[2];
    const int64_t R = p.requests;
    const int head = p.work[4 * R], free = p.work[4 * R + 1], all = p.starts[R];
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t t0 = (int64_t)blockIdx.x * 256, t = t0 + tid;
    int64_t r0 = 0, n = R;  // the requests that may have the workgroup's rows
    if (R > HELD && t0 < all) {
        if (tid < 128) {
            const int64_t r = request_of(p.starts, R, tid < 64 ? t0 : min(t0 + 255, (int64_t)all - 1));
            if (lane == 0) ends[tid >> 6] = r;
        }
        __syncthreads();
        r0 = ends[0];
        n = ends[1] - r0 + 1;
    }
    if (t0 < p.max_rows) {
#pragma unroll 8
        for (int64_t i = tid; i < min(n, (int64_t)HELD); i += 256) starts[i] = p.starts[r0 + i];
        __syncthreads();
    }
    if (t < all) {
        int64_t lo = 0, hi = n;
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if ((mid < HELD ? starts[mid] : p.starts[r0 + mid]) <= t)
                lo = mid;
            else
                hi = mid;
        }
        const work4 w = *(const work4 *)(p.work + 4 * (r0 + lo));
        fill_row(p, t, r0 + lo, w.x, w.y, w.z, head);
    }
    if (t >= all && t < p.max_rows) {
        p.slots[t] = -1;
        if (p.positions) p.positions[t] = 0;
    }
    give_back_all(p, (int64_t)blockIdx.x * 4 + (tid >> 6), (int64_t)gridDim.x * 4, head, free,
                  [&](int64_t r) {
                      const work4 w = *(const work4 *)(p.work + 4 * r);
                      return make_int4(w.x, w.y, w.z, w.w);
                  });
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

// A wave takes rows t0 .. t0 + 15 of 128 / D heads. T: the rows' type; STORE: into the pages, else out of them
// (bf16).
template <typename T, bool STORE, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void pages_rows_kernel(PageDims d, uint8_t *layer, T *k, T *v, int64_t k_row, int64_t k_head,
                                                         int64_t v_row, int64_t v_head, const int32_t *__restrict__ slots,
                                                         int64_t rows) {
    constexpr int OCT = D / 8, HEADS = 128 / D;      // lanes a row; heads of a wave
    __shared__ __attribute__((aligned(16))) uint8_t lds[WAVES][4096];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int h = (blockIdx.y * WAVES + wave) * HEADS + lane / (64 / HEADS);
    const int64_t t0 = (int64_t)blockIdx.x * 16;
    const int64_t most = d.pages * d.page_size;
    // lane i: the slot of row t0 - 15 + i, and whether it leads 16 rows with the slots of a granule
    const int64_t mine = t0 - 15 + lane;
    int slot = -1;
    if (lane < 46 && mine >= 0 && mine < rows) slot = slots[mine];
    if (slot < 0 || slot >= most) slot = -1;
    const uint64_t next = __ballot(slot >= 0 && __shfl_down(slot, 1) == slot + 1 && lane < 45);
    const uint64_t leads = __ballot(lane < 31 && slot >= 0 && (slot & 15) == 0 && ((next >> lane) & 0x7fffu) == 0x7fffu);
    const bool there = h < d.kv_heads;
    const int hs = there ? h : 0;
    auto granule = [&](int s) __attribute__((always_inline)) {
        const int page = s / d.page_size, in = s - page * d.page_size;
        return layer + (((int64_t)page * d.kv_heads + hs) * (d.page_size >> 4) + (in >> 4)) * granule_bytes(D);
    };

    const uint32_t here = (uint32_t)(leads >> 15) & 0xffffu;  // of rows t0 ..: at most one
    if (here) {
        const int lead = __builtin_ctz(here);
        const int64_t t = t0 + lead;
        uint8_t *g = granule(__builtin_amdgcn_readlane(slot, 15 + lead));
        // keys: 16 rows of four 16 B chunks a time (of each head 16 lanes a chunk)
        constexpr int CH = 4 / HEADS;
        const int l = lane % (64 / HEADS), key = l & 15;
        u32x4 y[OCT / CH];
#pragma unroll
        for (int i = 0; i < OCT / CH; i++) {
            const int c = i * CH + (l >> 4);
            T *src = k + (t + key) * k_row + hs * k_head + c * 8;
            if constexpr (STORE)
                y[i] = load8_bf16(src);
            else
                y[i] = *(const u32x4 *)(g + c * 256 + key * 16);
        }
        // values: four rows (a quad of keys) and eight dims a lane
        const int o = l % OCT, quad = l / OCT;
        uint8_t *const at = lds[wave] + lane / (64 / HEADS) * (4096 / HEADS);  // a head's granule half
        auto swap = [&](int dim) { return dim ^ ((dim >> 3) & 7); };            // (spreads the eight dims over the banks)
        u32x4 x[4];
        T *vp = v + (t + 4 * quad) * v_row + hs * v_head + o * 8;
        if constexpr (STORE) {
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = load8_bf16(vp + i * v_row);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int n = i * (64 / HEADS) + l, half = n / D, dim = n % D;
                *(u32x4 *)(at + half * (D * 16) + swap(dim) * 16) = *(const u32x4 *)(g + D * 32 + n * 16);
            }
        }
        if (there)
#pragma unroll
            for (int i = 0; i < OCT / CH; i++) {
                const int c = i * CH + (l >> 4);
                if constexpr (STORE)
                    *(u32x4 *)(g + c * 256 + key * 16) = y[i];
                else
                    *(u32x4 *)(k + (t + key) * k_row + hs * k_head + c * 8) = y[i];
            }
        uint8_t *const cell = at + (quad & 1) * (D * 16) + (quad >> 1) * 8;
        auto wait = [] {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        };
        if constexpr (STORE) {
#pragma unroll
            for (int e = 0; e < 8; e++) *(u32x2 *)(cell + swap(o * 8 + e) * 16) = column(x, e);
            wait();
            if (there)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int n = i * (64 / HEADS) + l, half = n / D, dim = n % D;
                    *(u32x4 *)(g + D * 32 + n * 16) = *(const u32x4 *)(at + half * (D * 16) + swap(dim) * 16);
                }
        } else {
            wait();
            u32x2 c[8];
#pragma unroll
            for (int e = 0; e < 8; e++) c[e] = *(const u32x2 *)(cell + swap(o * 8 + e) * 16);
            if (there)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t sel = i & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
                    for (int w = 0; w < 4; w++) x[i][w] = __builtin_amdgcn_perm(c[2 * w + 1][i >> 1], c[2 * w][i >> 1], sel);
                    *(u32x4 *)(vp + i * v_row) = x[i];
                }
        }
    }

    // the rows of no such 16, four at a time
    uint32_t rest = 0xffffu;
    for (uint64_t m = leads; m; m &= m - 1) {
        const int a = __builtin_ctzll(m) - 15;  // leads rows t0 + a .. a + 15
        rest &= ~(uint32_t)((a < 0 ? 0xffffull >> -a : 0xffffull << a));
    }
    if (rows - t0 < 16) rest &= (1u << (rows - t0)) - 1;
    if (!rest) return;
    const int o = lane % OCT, sub = lane % (64 / HEADS) / OCT;
    int at[4];
    u32x4 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = 4 * i + sub;
        at[i] = __shfl(slot, 15 + r);
        if (!there || !((rest >> r) & 1u)) at[i] = -2;
        x[i] = y[i] = u32x4{};
        if (at[i] < 0) continue;
        if constexpr (STORE) {
            x[i] = load8_bf16(k + (t0 + r) * k_row + h * k_head + o * 8);
            y[i] = load8_bf16(v + (t0 + r) * v_row + h * v_head + o * 8);
        } else {
            const uint8_t *g = granule(at[i]);
            x[i] = *(const u32x4 *)(g + granule_k(at[i] & 15, o * 8));
#pragma unroll
            for (int e = 0; e < 8; e++)
                y[i][e >> 1] |= (uint32_t)*(const uint16_t *)(g + granule_v(D, at[i] & 15, o * 8 + e)) << (16 * (e & 1));
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = 4 * i + sub;
        if constexpr (STORE) {
            if (at[i] < 0) continue;
            uint8_t *g = granule(at[i]);
            *(u32x4 *)(g + granule_k(at[i] & 15, o * 8)) = x[i];
#pragma unroll
            for (int e = 0; e < 8; e++)
                *(uint16_t *)(g + granule_v(D, at[i] & 15, o * 8 + e)) = (uint16_t)(y[i][e >> 1] >> (16 * (e & 1)));
        } else {
            if (at[i] < -1) continue;
            *(u32x4 *)(k + (t0 + r) * k_row + h * k_head + o * 8) = x[i];
            *(u32x4 *)(v + (t0 + r) * v_row + h * v_head + o * 8) = y[i];
        }
    }
}

template <typename T, bool STORE, int D>
hipError_t launch_heads(const PageDims &d, uint8_t *layer, T *k, T *v, int64_t k_row, int64_t k_head, int64_t v_row,
                        int64_t v_head, const int32_t *slots, int64_t rows, hipStream_t stream) {
    const int64_t blocks = (rows + 15) / 16, heads = (d.kv_heads + 128 / D - 1) / (128 / D);
    if (blocks >= (int64_t)1 << 24 || d.kv_heads > 65535) return hipErrorInvalidValue;
    // Workgroups of one wave as long as they do not fill the CUs: single tokens are a store of 64 lines after the
    // other (48 rows of 8 heads 5.0 us, 8.6 in fours).
    if (blocks * heads <= 4 * (int64_t)device_cu_count())
        pages_rows_kernel<T, STORE, D, 1><<<dim3((unsigned)blocks, (unsigned)heads), 64, 0, stream>>>(
            d, layer, k, v, k_row, k_head, v_row, v_head, slots, rows);
    else
        pages_rows_kernel<T, STORE, D, 4><<<dim3((unsigned)blocks, (unsigned)((heads + 3) / 4)), 256, 0, stream>>>(
            d, layer, k, v, k_row, k_head, v_row, v_head, slots, rows);
    return hipGetLastError();
}
template <typename T, bool STORE>
hipError_t launch_rows(const PageDims &d, uint8_t *layer, T *k, T *v, int64_t k_row, int64_t k_head, int64_t v_row,
                       int64_t v_head, const int32_t *slots, int64_t rows, hipStream_t stream) {
    if (rows <= 0) return hipSuccess;
    if (d.head_dim == 128) return launch_heads<T, STORE, 128>(d, layer, k, v, k_row, k_head, v_row, v_head, slots, rows, stream);
    if (d.head_dim == 64) return launch_heads<T, STORE, 64>(d, layer, k, v, k_row, k_head, v_row, v_head, slots, rows, stream);
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_page_plan(const PagePlanArgs &p, hipStream_t stream) {
    const int64_t blocks = (p.max_rows + 255) / 256;
    if (p.requests <= 0 || p.pages <= 0 || blocks >= (int64_t)1 << 24) return hipErrorInvalidValue;
    if (p.requests <= PLAN_REQUESTS && p.max_rows <= PLAN_ROWS) {
        if (p.requests <= 256 && p.max_rows <= 512)
            page_plan_kernel<256, true, 1><<<1, 256, 0, stream>>>(p);
        else
            page_plan_kernel<PLAN_REQUESTS, true, 1><<<1, PLAN_REQUESTS, 0, stream>>>(p);
        return hipGetLastError();
    }
    if (p.requests <= 4096)
        page_plan_kernel<1024, false, 4><<<1, 1024, 0, stream>>>(p);
    else
        page_plan_kernel<1024, false, 0><<<1, 1024, 0, stream>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // (a wave for every two requests, up to 4096 waves: all of those may be given back)
    page_fill_kernel<<<(unsigned)std::max(blocks, std::min((p.requests + 7) / 8, (int64_t)1024)), 256, 0, stream>>>(p);
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
