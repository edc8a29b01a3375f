// Low-rank adapters of many requests beside a shared projection (gfx950):
//   y[m] = x[m] W^T + scale_a (x[m] A_a^T) B_a^T,   a = ids[m] (none outside [0, n)).
//
// Two products: t = scale x A^T (ranks wide, K deep), then t B^T (N wide, ranks deep)
// added to the projection's f32 sums before the one rounding of y. Where the matrix pipe
// takes the second product t is the sum of bf16 numbers, each the rounding of what the ones
// before leave: two (2^-16 of t) for bf16 outputs, three (2^-24) for f32 ones, which keep the
// precision of their sums (with two 1.1e-6 instead of 2e-7 of 64 bits at 514 x 4096 x 4096).
//
// Rows of any adapters may lie next to each other: a tile of rows is multiplied once per
// adapter among its ids; of t the rows of other adapters are not written, in the second
// product they enter as zeros (adapters hold numbers only). Few rows are taken each by
// itself, so that many adapters are not multiplied one after the other. The second product
// of many rows runs as further k steps of the projection where that is over bf16 rows and not
// split over K (qgemm_bf16.hip), else as a pass over its f32 sums (lora_up_kernel).
#include <algorithm>
#include <type_traits>

#include "device_common.h"
#include "kernels.h"

namespace qimm {
namespace {

__device__ __forceinline__ int row_id(const int32_t *ids, int64_t row, int64_t m, int count) {
    if (row >= m) return -1;
    const int id = ids[row];
    return id >= 0 && id < count ? id : -1;
}

// ---- many rows: shares of K, 16 RT ranks at a time ----

// part[share][row][ldp] = x A^T over a share of K, for 128 rows and 16 RT ranks (from 64
// blockIdx.z) per workgroup, once per adapter among the rows' ids; rows of other adapters are
// not written. Bound by the bytes of x: both operands are copied HBM -> LDS by direct loads in
// whole 128 B rows of 64 deep (XOR-swizzled slots, three stages), since lanes that load their
// operand straight from 16 rows of x 64 B at a time reach half the bandwidth however many are
// in flight (4096 rows of 12288, 64 ranks: 46-52 us). A wave multiplies its 32 rows
// (v_mfma_f32_16x16x32_bf16, A = the adapter's rows; ranks past the last repeat it).
template <int RT>
__global__ __launch_bounds__(256, 2) void lora_down_kernel(const uint16_t *__restrict__ x, int64_t lda, int64_t m, int64_t K,
                                                          const AdapterDev *__restrict__ ad, int count,
                                                          const int32_t *__restrict__ ids, float *__restrict__ part, int64_t ldp) {
    constexpr int XB = 128 * 128, STAGE = XB + RT * 16 * 128;  // bytes of x rows and of a stage
    constexpr int AI = RT == 4 ? 2 : 1, NI = 4 + AI;           // direct loads of a wave and stage
    __shared__ __attribute__((aligned(16))) uint8_t lds[3 * STAGE];
    const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t tile0 = (int64_t)blockIdx.x * 128, row0 = tile0 + 32 * wave + l16;
    const int r0 = 64 * (int)blockIdx.z;
    const int64_t steps = K / 64, first = steps * blockIdx.y / gridDim.y, last = steps * (blockIdx.y + 1) / gridDim.y;
    part += (int64_t)blockIdx.y * m * ldp;
    const int id[2] = {row_id(ids, row0, m, count), row_id(ids, row0 + 16, m, count)};
    int all[2];  // of rows lane and lane + 64 of the tile
#pragma unroll
    for (int u = 0; u < 2; u++) {
        all[u] = row_id(ids, tile0 + 64 * u + lane, m, count);
        if (all[u] < 0) all[u] = 0x7fffffff;
    }
    uint32_t off[2];
#pragma unroll
    for (int ks = 0; ks < 2; ks++) off[ks] = (uint32_t)(l16 * 128 + (((4 * ks + lg) ^ swz_key(l16)) << 4));
    for (int a = -1;;) {
        // the next adapter of the tile: the smallest id above the last one
        int next = min(all[0] > a ? all[0] : 0x7fffffff, all[1] > a ? all[1] : 0x7fffffff);
        for (int o = 32; o > 0; o >>= 1) next = min(next, __shfl_xor(next, o));
        a = __builtin_amdgcn_readfirstlane(next);
        if (a == 0x7fffffff) break;
        const AdapterDev d = ad[a];
        if (r0 >= d.rank) continue;
        // one instruction fills 8 rows, lane l row l / 8 at slot l % 8, which holds chunk (l % 8) ^ key(row)
        const uint16_t *xs[4], *as[AI];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = 32 * wave + 8 * i + (lane >> 3);
            xs[i] = x + min(tile0 + r, m - 1) * lda + 8 * ((lane & 7) ^ swz_key(r));
        }
#pragma unroll
        for (int i = 0; i < AI; i++) {  // RT 1: two instructions, each issued by two waves
            const int r = (AI * wave + i) % (2 * RT) * 8 + (lane >> 3);
            as[i] = d.a + (int64_t)min(r0 + r, d.rank - 1) * K + 8 * ((lane & 7) ^ swz_key(r));
        }
        auto dma = [&](int s, int64_t step) __attribute__((always_inline)) {
            const int64_t k = min(step, last - 1) * 64;
#pragma unroll
            for (int i = 0; i < 4; i++)
                __builtin_amdgcn_global_load_lds((const void *)(xs[i] + k), (lds_ptr_t)(lds + s * STAGE + (32 * wave + 8 * i) * 128), 16, 0, 0);
#pragma unroll
            for (int i = 0; i < AI; i++)
                __builtin_amdgcn_global_load_lds((const void *)(as[i] + k),
                                                 (lds_ptr_t)(lds + s * STAGE + XB + (AI * wave + i) % (2 * RT) * 1024), 16, 0, 0);
        };
        f32x4 acc[2][RT] = {};
        dma(0, first);
        dma(1, first + 1);
        int s = 0;
        for (int64_t step = first; step < last; step++) {
            __builtin_amdgcn_s_waitcnt(WAIT_VM0 | NI);  // this step's rows have landed
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            dma(s == 0 ? 2 : s - 1, step + 2);  // the stage that the last step read
            const uint8_t *st = lds + s * STAGE;
            bf16x8 b[2][2], w[2][RT];
#pragma unroll
            for (int ks = 0; ks < 2; ks++) {
#pragma unroll
                for (int u = 0; u < 2; u++) b[ks][u] = *(const bf16x8 *)(st + (32 * wave + 16 * u) * 128 + off[ks]);
#pragma unroll
                for (int i = 0; i < RT; i++) w[ks][i] = *(const bf16x8 *)(st + XB + 16 * i * 128 + off[ks]);
            }
#pragma unroll
            for (int ks = 0; ks < 2; ks++)
#pragma unroll
                for (int i = 0; i < RT; i++)
#pragma unroll
                    for (int u = 0; u < 2; u++)
                        acc[u][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[ks][i], b[ks][u], acc[u][i], 0, 0, 0);
            s = s == 2 ? 0 : s + 1;
        }
        __builtin_amdgcn_s_waitcnt(WAIT_VM0_LGKM0);  // no load into LDS still in flight
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 2; u++)
            if (id[u] == a)
#pragma unroll
                for (int i = 0; i < RT; i++) *(f32x4 *)(part + (row0 + 16 * u) * ldp + r0 + 16 * i + 4 * lg) = acc[u][i];
    }
}

// four ranks' sums over the shares (stride apart), eight loads in flight
__device__ __forceinline__ f32x4 add_shares(const float *p, int shares, int64_t stride) {
    f32x4 s{};
    for (int i = 0; i < shares; i += 8) {
        f32x4 v[8];
#pragma unroll
        for (int u = 0; u < 8; u++) v[u] = *(const f32x4 *)(p + min(i + u, shares - 1) * stride);
#pragma unroll
        for (int u = 0; u < 8; u++)
            if (i + u < shares) s += v[u];
    }
    return s;
}
// the bf16 rounding of v (two in a word), and what it leaves
__device__ __forceinline__ uint32_t take_bf16x2(float &a, float &b) {
    const uint32_t w = pack_bf16x2(a, b);
    a -= __uint_as_float(w << 16);
    b -= __uint_as_float(w & 0xffff0000u);
    return w;
}

// The shares' sums times the scale as PARTS bf16 rows of `width` one after the other, zeros past
// the rank and up to ld; four ranks per thread. Rows without an adapter are not written. One
// after the other at the width of the ranks, not each from a step of 64 on: a tile of two
// adapters of rank 16 takes two k steps instead of four.
template <int PARTS>
__global__ __launch_bounds__(256) void lora_split_kernel(const float *__restrict__ part, int shares, int64_t m, int64_t ldp,
                                                        int64_t rows, const AdapterDev *__restrict__ ad, int count,
                                                        const int32_t *__restrict__ ids, uint16_t *__restrict__ t16, int64_t width,
                                                        int64_t ld) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = width / 4, row = i / per;
    if (row >= rows) return;
    const int id = row_id(ids, row, rows, count), r = (int)(i % per) * 4;
    if (id < 0) return;
    const int rank = ad[id].rank;
    const float scale = ad[id].scale;
    f32x4 s{};
    if (r < rank) s = add_shares(part + row * ldp + r, shares, m * ldp);  // written up to the rank's tile of 16
#pragma unroll
    for (int e = 0; e < 4; e++) s[e] = r + e < rank ? s[e] * scale : 0.f;
    uint16_t *dst = t16 + row * ld + r;
#pragma unroll
    for (int p = 0; p < PARTS; p++) {
        float a = s[0], b = s[1], c = s[2], d = s[3];
        *(u32x2 *)(dst + p * width) = u32x2{take_bf16x2(a, b), take_bf16x2(c, d)};
        s = f32x4{a, b, c, d};
    }
    for (int64_t e = PARTS * width; e + r < ld; e += width) *(u32x2 *)(dst + e) = u32x2{0, 0};
}

// y = base + t B^T for 16 rows x 256 columns, 64 columns per wave; t from the shares' sums,
// in PARTS bf16 operands. A = B's rows, B = t's. base: the product's sums, `splits` of them
// (base_stride apart) where it is split over K, added here in their order instead of in a
// launch of their own (514 rows x 4096 x 4096 BF16, rank 16: 48 -> 45 us in all). Bound by the
// bytes of base and y; the shares of t are read once per workgroup and go through LDS (each
// wave's own reads of up to 16 shares took 17 us at 1024 x 4096, now 12.7: 42 MB).
template <int PARTS>
__global__ __launch_bounds__(256) void lora_up_kernel(const float *__restrict__ part, int shares, int64_t m, int64_t ldp,
                                                     int64_t rows, int64_t N, const AdapterDev *__restrict__ ad, int count,
                                                     const int32_t *__restrict__ ids, const float *base, int splits,
                                                     int64_t base_stride, float *y32, uint16_t *y16) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
    // t of 32 ranks, each half of the workgroup the sum of every other share
    constexpr int PITCH = 36;
    __shared__ __attribute__((aligned(16))) float ts[2][16 * PITCH];
    const int half = tid >> 7, trow = (tid & 127) >> 3, tq = 4 * (tid & 7);
    const int64_t row0 = (int64_t)blockIdx.y * 16, row = row0 + l16;
    const int64_t n1 = (int64_t)blockIdx.x * 256 + 64 * wave, n0 = n1 < N ? n1 : 0;  // N is a multiple of 128
    const int id = row_id(ids, row, rows, count), tid_of = row_id(ids, row0 + trow, rows, count);
    f32x4 acc[4] = {}, base4[4];
#pragma unroll
    for (int i = 0; i < 4; i++) base4[i] = *(const f32x4 *)(base + min(row, rows - 1) * N + n0 + 16 * i + 4 * lg);
#pragma unroll 2
    for (int s = 1; s < splits; s++)
#pragma unroll
        for (int i = 0; i < 4; i++) base4[i] += *(const f32x4 *)(base + s * base_stride + min(row, rows - 1) * N + n0 + 16 * i + 4 * lg);
    uint64_t todo = __ballot(id >= 0) & 0xffffu;
    while (todo) {
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
        todo &= ~__ballot(id == a);
        const AdapterDev d = ad[a];
        for (int r0 = 0; r0 < d.rank; r0 += 32) {
            const int r = r0 + 8 * lg;
            f32x4 t4{};
            if (tid_of == a && r0 + tq < d.rank)
                t4 = add_shares(part + half * (m * ldp) + (row0 + trow) * ldp + r0 + tq, (shares - half + 1) / 2, 2 * m * ldp);
            __syncthreads();
            *(f32x4 *)&ts[half][trow * PITCH + tq] = t4;
            __syncthreads();
            const float *t0 = &ts[0][l16 * PITCH + 8 * lg], *t1 = &ts[1][l16 * PITCH + 8 * lg];
            f32x4 u = *(const f32x4 *)t0 + *(const f32x4 *)t1, v = *(const f32x4 *)(t0 + 4) + *(const f32x4 *)(t1 + 4);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                u[e] = r + e < d.rank ? u[e] * d.scale : 0.f;
                v[e] = r + 4 + e < d.rank ? v[e] * d.scale : 0.f;
            }
            bf16x8 b[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                b[i] = bf16x8{};
                if (r < d.ldb) b[i] = *(const bf16x8 *)(d.b + (n0 + 16 * i + l16) * d.ldb + r);
            }
#pragma unroll
            for (int p = 0; p < PARTS; p++) {
                float t[8] = {u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
                const u32x4 w = u32x4{take_bf16x2(t[0], t[1]), take_bf16x2(t[2], t[3]), take_bf16x2(t[4], t[5]), take_bf16x2(t[6], t[7])};
                u = f32x4{t[0], t[1], t[2], t[3]};
                v = f32x4{t[4], t[5], t[6], t[7]};
#pragma unroll
                for (int i = 0; i < 4; i++)
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[i], __builtin_bit_cast(bf16x8, w), acc[i], 0, 0, 0);
            }
        }
    }
    if (row >= rows || n1 >= N) return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int64_t at = row * N + n0 + 16 * i + 4 * lg;
        const f32x4 s = base4[i] + acc[i];
        if (y32)
            *(f32x4 *)(y32 + at) = s;
        else
            *(u32x2 *)(y16 + at) = u32x2{pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3])};
    }
}

// ---- few rows: every row by itself ----

__device__ __forceinline__ float dot8(u32x4 a, u32x4 b, float s) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        s = __builtin_fmaf(__uint_as_float(a[e] << 16), __uint_as_float(b[e] << 16), s);
        s = __builtin_fmaf(__uint_as_float(a[e] & 0xffff0000u), __uint_as_float(b[e] & 0xffff0000u), s);
    }
    return s;
}

// t of row blockIdx.y, one rank per wave.
__global__ __launch_bounds__(256) void lora_down_row_kernel(const uint16_t *__restrict__ x, int64_t lda, int64_t K,
                                                           const AdapterDev *__restrict__ ad, int count,
                                                           const int32_t *__restrict__ ids, float *__restrict__ t, int64_t ldt) {
    const int64_t row = blockIdx.y;
    const int id = ids[row];
    if (id < 0 || id >= count) return;
    const AdapterDev d = ad[id];
    const int lane = threadIdx.x & 63, r = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (r >= d.rank) return;
    const uint16_t *xr = x + row * lda, *ar = d.a + (int64_t)r * K;
    float s[4] = {0.f, 0.f, 0.f, 0.f};  // four chains: a row's loads are all in flight at once
    int64_t k = 8 * lane;
    for (; k + 3 * 512 < K; k += 4 * 512) {
#pragma unroll
        for (int u = 0; u < 4; u++) s[u] = dot8(*(const u32x4 *)(xr + k + 512 * u), *(const u32x4 *)(ar + k + 512 * u), s[u]);
    }
    for (; k < K; k += 512) s[0] = dot8(*(const u32x4 *)(xr + k), *(const u32x4 *)(ar + k), s[0]);
    const float sum = wave_sum((s[0] + s[1]) + (s[2] + s[3]));
    if (lane == 0) t[row * ldt + r] = sum * d.scale;
}

// y of row blockIdx.y, one column per thread: a thread reads its row of B, 16 B at a time.
__global__ __launch_bounds__(256) void lora_up_row_kernel(const float *__restrict__ t, int64_t ldt, int64_t N,
                                                         const AdapterDev *__restrict__ ad, int count,
                                                         const int32_t *__restrict__ ids, const float *base, int splits,
                                                         int64_t base_stride, float *y32, uint16_t *y16) {
    const int64_t row = blockIdx.y, n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int id = ids[row];
    if (n >= N) return;
    float b0 = base[row * N + n];
    for (int s = 1; s < splits; s++) b0 += base[s * base_stride + row * N + n];
    float s = 0.f;
    if (id >= 0 && id < count) {
        const AdapterDev d = ad[id];
        const float *tr = t + row * ldt;
        const uint16_t *br = d.b + n * d.ldb;
        for (int r = 0; r < d.rank; r += 8) {
            const u32x4 b = *(const u32x4 *)(br + r);  // zeros past the rank, where t is not written
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (r + e < d.rank)
                    s = __builtin_fmaf(tr[r + e], __uint_as_float(e & 1 ? b[e >> 1] & 0xffff0000u : b[e >> 1] << 16), s);
        }
    }
    s += b0;
    if (y32)
        y32[row * N + n] = s;
    else
        y16[row * N + n] = (uint16_t)(pack_bf16x2(s, 0.f) & 0xffffu);
}

__global__ __launch_bounds__(256) void repeat_ids_kernel(const int32_t *__restrict__ ids, int64_t rows, int64_t per,
                                                        int32_t *__restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < rows) out[i] = ids[i / per];
}

// Each row is taken by itself up to 64 rows, and up to 256 of small ranks: the tiles' time grows with
// the adapters among their rows, of which the host knows only how many are held. us, by tiles with one
// adapter / one per row -> by rows, the same: Q8_0 4096 x 4096, rank 16, 64 rows 24 / 155 -> 22 / 22,
// 128 rows 29 / 277 -> 27 / 27, 256 rows 32 / 284 -> 32 / 38; rank 64, 64 rows 27 / 229 -> 26 / 43, 128
// rows 31 / 389 -> 34 / 92, 256 rows 36 / 435 -> 50 / 165. Q4_K 12288 x 4096, rank 64, 64 rows 32 / 235 ->
// 50 / 127, 128 rows 45 / 453 -> 80 / 242, 256 rows 52 / 494 -> 123 / 453; rank 1024 (16 adapters), 16 rows
// 77 / 993 -> 115 / 163, 64 rows 87 / 999 -> 425 / 1239. So it gives away: large ranks of one adapter at up
// to 64 rows, 128 rows of one of eight or more adapters held, and, by tiles, more than 128 rows of rank 64
// with an adapter each.
constexpr int64_t FEW_ROWS = 64, MORE_ROWS = 256;

}  // namespace

hipError_t launch_repeat_ids(const int32_t *ids, int64_t rows, int64_t per, int32_t *out, hipStream_t stream) {
    if (rows <= 0) return hipSuccess;
    repeat_ids_kernel<<<dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, stream>>>(ids, rows, per, out);
    return hipGetLastError();
}

bool lora_few(int64_t m, int64_t max_rank, int64_t count) {
    return m <= FEW_ROWS || (m <= MORE_ROWS && m * max_rank <= (count >= 8 ? 8192 : 4096));
}

hipError_t launch_lora_few_down(const uint16_t *x, int64_t lda, int64_t m, int64_t k, const AdapterDev *ad, int count,
                                const int32_t *ids, float *t, int64_t ldt, hipStream_t stream) {
    if (m <= 0) return hipSuccess;
    if (m > MORE_ROWS) return hipErrorInvalidValue;
    lora_down_row_kernel<<<dim3((unsigned)((ldt + 3) / 4), (unsigned)m), dim3(256), 0, stream>>>(x, lda, k, ad, count, ids, t, ldt);
    return hipGetLastError();
}

hipError_t launch_lora_few_up(const float *t, int64_t ldt, int64_t m, int64_t n, const AdapterDev *ad, int count,
                              const int32_t *ids, SplitSums base, float *y32, uint16_t *y16, hipStream_t stream) {
    if (m <= 0) return hipSuccess;
    if (m > MORE_ROWS) return hipErrorInvalidValue;
    lora_up_row_kernel<<<dim3((unsigned)((n + 255) / 256), (unsigned)m), dim3(256), 0, stream>>>(t, ldt, n, ad, count, ids, base.part,
                                                                                                base.splits, m * n, y32, y16);
    return hipGetLastError();
}

// Ranks per workgroup: 16, 32 or 64 at a time; shares of K: as many as give every CU two
// workgroups, each of at least 4 steps of 64, and at most 16 (the second product adds them:
// 48 shares of 12288 at 1024 rows took it 29 us).
namespace {
int rank_tile(int64_t max_rank) { return max_rank <= 16 ? 16 : max_rank <= 32 ? 32 : 64; }
int down_shares(int64_t m, int64_t k, int64_t max_rank) {
    const int64_t rt = rank_tile(max_rank), wgs = (m + 127) / 128 * ((max_rank + rt - 1) / rt);
    return (int)std::max<int64_t>(1, std::min<int64_t>({2 * std::max(device_cu_count(), 1) / wgs, k / 256, 16}));
}
}  // namespace

LoraShares lora_shares(int64_t m, int64_t k, int64_t max_rank) {
    const int64_t rt = rank_tile(max_rank);
    return {down_shares(m, k, max_rank), (max_rank + rt - 1) / rt * rt};
}

size_t lora_down_scratch(int64_t m, int64_t k, int64_t max_rank) {
    const LoraShares s = lora_shares(m, k, max_rank);
    return (size_t)(s.shares * m * s.ldp) * 4;
}

hipError_t launch_lora_down(const uint16_t *x, int64_t lda, int64_t m, int64_t k, int64_t max_rank, const AdapterDev *ad, int count,
                            const int32_t *ids, float *part, hipStream_t stream) {
    if (m <= 0) return hipSuccess;
    const int64_t rt = rank_tile(max_rank);
    const LoraShares s = lora_shares(m, k, max_rank);
    const dim3 grid((unsigned)((m + 127) / 128), (unsigned)s.shares, (unsigned)(s.ldp / rt));
    if (rt == 16)
        lora_down_kernel<1><<<grid, dim3(256), 0, stream>>>(x, lda, m, k, ad, count, ids, part, s.ldp);
    else if (rt == 32)
        lora_down_kernel<2><<<grid, dim3(256), 0, stream>>>(x, lda, m, k, ad, count, ids, part, s.ldp);
    else
        lora_down_kernel<4><<<grid, dim3(256), 0, stream>>>(x, lda, m, k, ad, count, ids, part, s.ldp);
    return hipGetLastError();
}

hipError_t launch_lora_split(const float *part, LoraShares sh, int64_t m, int64_t width, int parts, const AdapterDev *ad, int count,
                             const int32_t *ids, uint16_t *t16, int64_t ld, hipStream_t stream) {
    if (m <= 0) return hipSuccess;
    if ((parts != 2 && parts != 3) || width % 8 || ld % 8 || ld < parts * width) return hipErrorInvalidValue;
    constexpr int64_t MOST = 1 << 20;  // rows of one grid (2^28 threads at rank 1024)
    for (int64_t r = 0; r < m; r += MOST) {
        const int64_t rows = std::min(m - r, MOST);
        const dim3 grid((unsigned)((rows * (width / 4) + 255) / 256));
        const float *p = part + r * sh.ldp;
        uint16_t *t = t16 + r * ld;
        if (parts == 2)
            lora_split_kernel<2><<<grid, dim3(256), 0, stream>>>(p, sh.shares, m, sh.ldp, rows, ad, count, ids + r, t, width, ld);
        else
            lora_split_kernel<3><<<grid, dim3(256), 0, stream>>>(p, sh.shares, m, sh.ldp, rows, ad, count, ids + r, t, width, ld);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_lora_up(const float *part, LoraShares sh, int64_t m, int64_t row0, int64_t rows, int64_t n, const AdapterDev *ad,
                          int count, const int32_t *ids, SplitSums base, float *y32, uint16_t *y16, hipStream_t stream) {
    if (n % 128) return hipErrorInvalidValue;
    constexpr int64_t MOST = 16 * 65535;  // rows of one grid
    for (int64_t r = 0; r < rows; r += MOST) {
        const int64_t some = std::min(rows - r, MOST);
        const dim3 grid((unsigned)((n + 255) / 256), (unsigned)((some + 15) / 16));
        const float *p = part + (row0 + r) * sh.ldp;
        if (y32)
            lora_up_kernel<3><<<grid, dim3(256), 0, stream>>>(p, sh.shares, m, sh.ldp, some, n, ad, count, ids + r, base.part + r * n,
                                                             base.splits, rows * n, y32 + r * n, nullptr);
        else
            lora_up_kernel<2><<<grid, dim3(256), 0, stream>>>(p, sh.shares, m, sh.ldp, some, n, ad, count, ids + r, base.part + r * n,
                                                             base.splits, rows * n, nullptr, y16 + r * n);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace qimm
