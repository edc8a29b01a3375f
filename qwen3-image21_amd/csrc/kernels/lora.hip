// Low-rank adapters of many requests beside a shared projection (gfx950):
//   y[m] = x[m] W^T + scale_a (x[m] A_a^T) B_a^T,   a = ids[m] (none outside [0, n)).
//
// Two products: t = scale x A^T (ranks wide, K deep), then t B^T (N wide, ranks deep)
// added to the projection's f32 sums before the one rounding of y. t is held in f32 and
// enters the second product as the sum of two bf16 numbers, hi = bf16(t) and lo = bf16(t -
// hi): 2^-17 of t, so that f32 outputs keep the precision of their sums.
//
// Rows of any adapters may lie next to each other: a tile of 16 rows is multiplied once per
// adapter among its ids; of t the rows of other adapters are not written, in the second
// product they enter as zeros.
#include <algorithm>

#include "device_common.h"
#include "kernels.h"

namespace qimm {
namespace {

__device__ __forceinline__ int row_id(const int32_t *ids, int64_t row, int64_t m, int count) {
    if (row >= m) return -1;
    const int id = ids[row];
    return id >= 0 && id < count ? id : -1;
}

// t[row][0 .. 32 ceil(rank / 32)) for a tile of 16 rows; the four waves share K, 64 ranks at
// a time. A = the adapter's rows (ranks past the last repeat it, their sums become 0), B = x.
__global__ __launch_bounds__(256) void lora_down_kernel(const uint16_t *__restrict__ x, int64_t lda, int64_t m, int64_t K,
                                                       const AdapterDev *__restrict__ ad, int count,
                                                       const int32_t *__restrict__ ids, float *__restrict__ t, int64_t ldt) {
    __shared__ f32x4 red[4][4][64];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
    const int64_t row = (int64_t)blockIdx.x * 16 + l16;
    const int id = row_id(ids, row, m, count);
    const uint16_t *xr = x + min(row, m - 1) * lda + 8 * lg;
    uint64_t todo = __ballot(id >= 0) & 0xffffu;
    while (todo) {
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
        todo &= ~__ballot(id == a);
        const AdapterDev d = ad[a];
        for (int r0 = 0; r0 < d.rank; r0 += 64) {
            f32x4 acc[4] = {};
            const uint16_t *ar[4];
#pragma unroll
            for (int i = 0; i < 4; i++) ar[i] = d.a + (int64_t)min(r0 + 16 * i + l16, d.rank - 1) * K + 8 * lg;
            for (int64_t k = 32 * wave; k < K; k += 128) {
                const bf16x8 b = *(const bf16x8 *)(xr + k);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8 *)(ar[i] + k), b, acc[i], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) red[wave][i][lane] = acc[i];
            __syncthreads();
            // wave i adds rank tile i: ranks r0 + 16 i + 4 lg + e of token l16
            f32x4 s = red[0][wave][lane];
#pragma unroll
            for (int w = 1; w < 4; w++) s += red[w][wave][lane];
            const int r = r0 + 16 * wave + 4 * lg;
#pragma unroll
            for (int e = 0; e < 4; e++) s[e] = r + e < d.rank ? s[e] * d.scale : 0.f;
            if (id == a && r < ((d.rank + 31) & ~31)) *(f32x4 *)(t + row * ldt + r) = s;
            __syncthreads();
        }
    }
}

// y = base + t B^T for 16 rows x 256 columns, 64 columns per wave. A = B's rows, B = t.
__global__ __launch_bounds__(256) void lora_up_kernel(const float *__restrict__ t, int64_t ldt, int64_t m, int64_t N,
                                                     const AdapterDev *__restrict__ ad, int count,
                                                     const int32_t *__restrict__ ids, const float *base,
                                                     float *y32, uint16_t *y16) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
    const int64_t row = (int64_t)blockIdx.y * 16 + l16, n0 = (int64_t)blockIdx.x * 256 + 64 * wave;
    if (n0 >= N) return;  // N is a multiple of 128
    const int id = row_id(ids, row, m, count);
    f32x4 acc[4] = {};
    uint64_t todo = __ballot(id >= 0) & 0xffffu;
    while (todo) {
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
        todo &= ~__ballot(id == a);
        const AdapterDev d = ad[a];
        for (int r0 = 0; r0 < d.rank; r0 += 32) {
            const int r = r0 + 8 * lg;
            f32x4 u{}, v{};
            if (id == a) {
                u = *(const f32x4 *)(t + row * ldt + r);
                v = *(const f32x4 *)(t + row * ldt + r + 4);
            }
            const u32x4 hi = u32x4{pack_bf16x2(u[0], u[1]), pack_bf16x2(u[2], u[3]), pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
            u32x4 lo;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float p = e < 2 ? u[2 * e] : v[2 * e - 4], q = e < 2 ? u[2 * e + 1] : v[2 * e - 3];
                lo[e] = pack_bf16x2(p - __uint_as_float(hi[e] << 16), q - __uint_as_float(hi[e] & 0xffff0000u));
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                u32x4 b{};
                if (r < d.ldb) b = *(const u32x4 *)(d.b + (n0 + 16 * i + l16) * d.ldb + r);
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, hi), acc[i], 0, 0, 0);
                acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, lo), acc[i], 0, 0, 0);
            }
        }
    }
    if (row >= m) return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int64_t at = row * N + n0 + 16 * i + 4 * lg;
        const f32x4 s = *(const f32x4 *)(base + at) + acc[i];
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
                                                         const int32_t *__restrict__ ids, const float *base, float *y32,
                                                         uint16_t *y16) {
    const int64_t row = blockIdx.y, n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int id = ids[row];
    if (n >= N) return;
    const float b0 = base[row * N + n];
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

// Up to this many rows each row is taken by itself.
constexpr int64_t FEW_ROWS = 64;

}  // namespace

hipError_t launch_lora_down(const uint16_t *x, int64_t lda, int64_t m, int64_t k, const AdapterDev *ad, int count,
                            const int32_t *ids, float *t, int64_t ldt, hipStream_t stream) {
    if (m <= 0) return hipSuccess;
    if (m <= FEW_ROWS) {
        lora_down_row_kernel<<<dim3((unsigned)((ldt + 3) / 4), (unsigned)m), dim3(256), 0, stream>>>(x, lda, k, ad, count, ids, t, ldt);
        return hipGetLastError();
    }
    lora_down_kernel<<<dim3((unsigned)((m + 15) / 16)), dim3(256), 0, stream>>>(x, lda, m, k, ad, count, ids, t, ldt);
    return hipGetLastError();
}

hipError_t launch_lora_up(const float *t, int64_t ldt, int64_t m, int64_t n, const AdapterDev *ad, int count,
                          const int32_t *ids, const float *base, float *y32, uint16_t *y16, hipStream_t stream) {
    if (m <= 0) return hipSuccess;
    if (n % 128 || (m + 15) / 16 > 65535) return hipErrorInvalidValue;
    if (m <= FEW_ROWS) {
        lora_up_row_kernel<<<dim3((unsigned)((n + 255) / 256), (unsigned)m), dim3(256), 0, stream>>>(t, ldt, n, ad, count, ids,
                                                                                                    base, y32, y16);
        return hipGetLastError();
    }
    lora_up_kernel<<<dim3((unsigned)((n + 255) / 256), (unsigned)((m + 15) / 16)), dim3(256), 0, stream>>>(t, ldt, m, n, ad, count,
                                                                                                          ids, base, y32, y16);
    return hipGetLastError();
}

}  // namespace qimm
