// The prefix cache held in 4 bits: storing a layer, and reading it back as bf16
// (gfx950). The format is in kv4.h.
//
// A block of values x stands for the nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} 2^s,
// ties to the even code, with s the smallest integer for which max|x| <= 7 2^s (the
// largest value is then off by at most half the spacing at the top of the range), within
// [-120, 125]. s comes from the exponent and the mantissa of the largest magnitude, an
// integer comparison; the codes and the values from the hardware's conversions, which
// round once, by a power of two: the same bits on every path.
//
// What bounds it: bytes. Storing reads 2 B a value and writes 4.25 bits, reading back the
// other way round. 16 B accesses, one block per thread and step; V is taken from rows
// [P][128] by threads that hold four dimensions of 32 keys, so that rows are read 256 B
// at a time.
#include <algorithm>

#include "kernels.h"
#include "kv4.h"

namespace qimm {
namespace {

// the scale byte of a block whose largest magnitude has these bf16 bits (a number)
__device__ __forceinline__ uint32_t scale_byte(uint32_t mag) {
    const int s = (int)(mag >> 7) - ((mag & 127u) <= 96u ? 2 : 1);  // mantissa 1 + 96 / 128 = 7 / 4
    return (uint32_t)min(max(s, 127 - 120), 127 + 125);
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

__device__ __forceinline__ uint32_t max_mag(uint32_t a, uint32_t w) {
    return max(a, max(w & 0x7fffu, (w >> 16) & 0x7fffu));
}

// four codes pairs from four words of two bf16 each
__device__ __forceinline__ uint32_t encode8(u32x4 w, float sc) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (uint32_t)w[0]), sc, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (uint32_t)w[1]), sc, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (uint32_t)w[2]), sc, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (uint32_t)w[3]), sc, 3);
    return r;
}
__device__ __forceinline__ u32x4 decode8(uint32_t c, float sc) {
    u32x4 r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 3));
    return r;
}

__device__ __forceinline__ int chunk_of(int base, int i, int lane) { return base + (i * 64 + lane) * 16; }
__device__ __forceinline__ int scale_at(int base, int i, int lane) { return base + ((i >> 2) * 64 + lane) * 4 + (i & 3); }

// ---- storing ----

// Keys [BH][P][128] (bf16), one block of 32 dimensions per thread and step, the tiles in turn
// over the workgroups. A block with a NaN or an infinity gets the scale byte 255 and stands for
// NaN throughout: the key's scores are NaN, as they would be from the bf16 cache. A key with
// kvalid[b][key] == 0 is stored as zeros. part[workgroup]: the largest norm of its keys; the
// kernel that stores the values comes after this one and takes their maximum (an atomic
// maximum of every tile into one address took 5-10 ns each: 8395 keys of 32 heads 36 us).
__global__ __launch_bounds__(256) void store_k4_kernel(const uint16_t *__restrict__ k, int64_t P, int64_t heads,
                                                       const uint8_t *__restrict__ kvalid, int64_t valid_ld, int64_t T,
                                                       int64_t count, uint8_t *__restrict__ tiles, float *__restrict__ part) {
    __shared__ float top[4];
    __shared__ __attribute__((aligned(16))) uint8_t scales[512];
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
    float most = 0.f;
    for (int64_t at = blockIdx.x; at < count; at += gridDim.x) {
        const int64_t bh = at / T, t = at % T;
        uint8_t *tile = tiles + at * KV4_TILE;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int i = (tid >> 6) + 4 * h;
            const int64_t key = t * KV4_KEYS + kv4_key(i, l16);
            u32x4 w[4] = {};
            if (key < P && (!kvalid || kvalid[bh / heads * valid_ld + key])) {
                const u32x4 *src = (const u32x4 *)(k + (bh * P + key) * 128 + 32 * lg);
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = src[e];
            }
            uint32_t mag = 0;
#pragma unroll
            for (int e = 0; e < 16; e++) mag = max_mag(mag, w[e >> 2][e & 3]);
            const uint32_t byte = mag < 0x7f80u ? scale_byte(mag) : 255u;
            const float sc = scale_of(mag < 0x7f80u ? byte : 127u);
            u32x4 c;
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                c[e] = encode8(w[e], sc);
                const u32x4 v = decode8(c[e], sc);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const float a = __uint_as_float(v[q] << 16), b = __uint_as_float(v[q] & 0xffff0000u);
                    ss += a * a + b * b;
                }
            }
            if (byte == 255u) ss = INFINITY;
            *(u32x4 *)(tile + chunk_of(0, i, lane)) = c;
            scales[scale_at(0, i, lane)] = (uint8_t)byte;
            ss += __shfl_xor(ss, 16);
            ss += __shfl_xor(ss, 32);
            most = fmaxf(most, ss);
        }
        __syncthreads();
        if (tid < 32) *(u32x4 *)(tile + KV4_KS + 16 * tid) = *(const u32x4 *)(scales + 16 * tid);
        __syncthreads();
    }
    for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    if (lane == 0) top[tid >> 6] = most;
    __syncthreads();
    // a bound: the f32 sum of 128 squares and the root are off by less than 2^-16
    if (tid == 0) part[blockIdx.x] = sqrtf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]))) * 1.0001f;
}

// the maximum of store_k4_kernel's parts, by one workgroup of the kernel launched after it
__device__ __forceinline__ void join_norms(const float *part, int parts, float *norm) {
    __shared__ float top[4];
    float most = 0.f;
    for (int i = threadIdx.x; i < parts; i += 256) most = fmaxf(most, part[i]);
    for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = most;
    __syncthreads();
    if (threadIdx.x == 0) *norm = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}

// One block of values: its scale byte, and the codes. 32 keys share it, so a value that is
// no number must not spoil the others (its key may be one that a mask hides): a NaN counts
// as 0, an infinity as the largest that the block's numbers allow.
__device__ __forceinline__ u32x4 encode_v(u32x4 (&w)[4], uint32_t &byte) {
    uint32_t mag = 0;
#pragma unroll
    for (int e = 0; e < 16; e++) mag = max_mag(mag, w[e >> 2][e & 3]);
    if (__builtin_expect(mag >= 0x7f80u, 0)) {
        mag = 0;
        uint32_t inf = 0;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            uint32_t x = w[e >> 2][e & 3];
            if ((x & 0x7fffu) > 0x7f80u) x &= 0xffff0000u;
            if (((x >> 16) & 0x7fffu) > 0x7f80u) x &= 0xffffu;
            w[e >> 2][e & 3] = x;
            const uint32_t lo = x & 0x7fffu, hi = (x >> 16) & 0x7fffu;
            if (lo < 0x7f80u) mag = max(mag, lo); else inf = 1;
            if (hi < 0x7f80u) mag = max(mag, hi); else inf = 1;
        }
        byte = scale_byte(mag);
        if (inf)  // +-6 2^s, which the conversion keeps
#pragma unroll
            for (int e = 0; e < 16; e++) {
                uint32_t x = w[e >> 2][e & 3];
                const uint32_t six = __float_as_uint(6.0f * scale_of(byte)) >> 16;
                if ((x & 0x7fffu) == 0x7f80u) x = (x & 0xffff8000u) | six;
                if (((x >> 16) & 0x7fffu) == 0x7f80u) x = (x & 0x8000ffffu) | (six << 16);
                w[e >> 2][e & 3] = x;
            }
    } else {
        byte = scale_byte(mag);
    }
    const float sc = scale_of(byte);
    u32x4 c;
#pragma unroll
    for (int e = 0; e < 4; e++) c[e] = encode8(w[e], sc);
    return c;
}

// Values [BH][P][128] (bf16): a thread holds four dimensions of 32 keys, a workgroup two tiles.
__global__ __launch_bounds__(256) void store_v4_kernel(const uint16_t *__restrict__ v, int64_t P, int64_t T,
                                                       uint8_t *__restrict__ tiles, const float *__restrict__ part,
                                                       int parts, float *__restrict__ norm) {
    __shared__ __attribute__((aligned(16))) uint8_t scales[2][512];
    const int half = threadIdx.x >> 7;
    const int64_t bh = blockIdx.y, t = (int64_t)blockIdx.x * 2 + half;
    if (blockIdx.x == 0 && bh == 0) join_norms(part, parts, norm);
    const int d4 = threadIdx.x & 31, lg = (threadIdx.x >> 5) & 3;
    const int64_t key0 = t * KV4_KEYS + 32 * lg;
    const uint16_t *src = v + (bh * P + key0) * 128 + 4 * d4;
    u32x2 r[32];
    if (key0 + 32 <= P) {
#pragma unroll
        for (int n = 0; n < 32; n++) r[n] = *(const u32x2 *)(src + n * 128);
    } else {
#pragma unroll
        for (int n = 0; n < 32; n++) r[n] = key0 + n < P ? *(const u32x2 *)(src + n * 128) : u32x2{0, 0};
    }
    uint8_t *tile = tiles + (bh * T + t) * KV4_TILE;
#pragma unroll
    for (int d = 0; d < 4; d++) {
        u32x4 w[4];
#pragma unroll
        for (int e = 0; e < 16; e++)  // the halves of two keys' words
            w[e >> 2][e & 3] = __builtin_amdgcn_perm(r[2 * e + 1][d >> 1], r[2 * e][d >> 1], d & 1 ? 0x07060302u : 0x05040100u);
        uint32_t byte;
        const u32x4 c = encode_v(w, byte);
        const int dim = 4 * d4 + d, j = dim >> 4, lane = 16 * lg + (dim & 15);
        if (t < T) *(u32x4 *)(tile + chunk_of(KV4_V, j, lane)) = c;
        scales[half][scale_at(0, j, lane)] = (uint8_t)byte;
    }
    __syncthreads();
    const int q = threadIdx.x & 127;
    if (t < T && q < 32) *(u32x4 *)(tile + KV4_VS + 16 * q) = *(const u32x4 *)(scales[half] + 16 * q);
}

// Values already transposed, vt [BH][128][ld] (ld a multiple of 8): one block per thread and step.
__global__ __launch_bounds__(256) void store_vt4_kernel(const uint16_t *__restrict__ vt, int64_t ld, int64_t P,
                                                        int64_t heads, const uint8_t *__restrict__ kvalid,
                                                        int64_t valid_ld, uint8_t *__restrict__ tiles,
                                                        const float *__restrict__ part, int parts, float *__restrict__ norm) {
    const int64_t bh = blockIdx.y, T = gridDim.x;
    if (blockIdx.x == 0 && bh == 0) join_norms(part, parts, norm);
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
    uint8_t *tile = tiles + (bh * T + blockIdx.x) * KV4_TILE;
    const int64_t key0 = (int64_t)blockIdx.x * KV4_KEYS + 32 * lg;
    uint32_t keep = 0;  // bit n: key key0 + n exists and is valid
#pragma unroll
    for (int n = 0; n < 32; n++)
        if (key0 + n < P && (!kvalid || kvalid[bh / heads * valid_ld + key0 + n])) keep |= 1u << n;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int j = (tid >> 6) + 4 * h;
        const uint16_t *src = vt + (bh * 128 + 16 * j + l16) * ld + key0;
        u32x4 w[4] = {};
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (key0 + 8 * e < P) w[e] = *(const u32x4 *)(src + 8 * e);  // within the row: ld >= P rounded up to 8
#pragma unroll
        for (int e = 0; e < 16; e++)
            w[e >> 2][e & 3] &= ((keep >> (2 * e)) & 1u ? 0xffffu : 0u) | ((keep >> (2 * e + 1)) & 1u ? 0xffff0000u : 0u);
        uint32_t byte;
        const u32x4 c = encode_v(w, byte);
        *(u32x4 *)(tile + chunk_of(KV4_V, j, lane)) = c;
        tile[scale_at(KV4_VS, j, lane)] = (uint8_t)byte;
    }
}

// ---- reading back ----

// bf16 K [BH][P][128] and, with VT, V^T [BH][128][ld] (the attention's layouts), else V
// [BH][P][128]; one tile per workgroup, blockIdx.z 0: K, 1: V.
template <bool VT>
__global__ __launch_bounds__(256) void load4_kernel(const uint8_t *__restrict__ tiles, int64_t P, int64_t ld,
                                                    uint16_t *__restrict__ k, uint16_t *__restrict__ v) {
    const int64_t bh = blockIdx.y, T = gridDim.x;
    const int tid = threadIdx.x;
    const uint8_t *tile = tiles + (bh * T + blockIdx.x) * KV4_TILE;
    const int64_t first = (int64_t)blockIdx.x * KV4_KEYS;
    // 16 B of the output per thread and step, 16 threads a row of 256 B: eight dimensions of
    // a key or, transposed, eight keys of a dimension, one word of codes
    if (blockIdx.z == 0) {
#pragma unroll
        for (int h = 0; h < 8; h++) {
            const int at = (tid >> 4) + 16 * h, piece = tid & 15;  // key of the tile
            const int i = 4 * (at >> 6) + ((at >> 2) & 3), lane = 16 * (piece >> 2) + 4 * ((at >> 4) & 3) + (at & 3);
            if (first + at >= P) continue;
            const uint32_t c = *(const uint32_t *)(tile + chunk_of(0, i, lane) + 4 * (piece & 3));
            const uint32_t byte = tile[scale_at(KV4_KS, i, lane)];
            *(u32x4 *)(k + (bh * P + first + at) * 128 + 8 * piece) =
                byte == 255u ? u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u} : decode8(c, scale_of(byte));
        }
    } else if constexpr (VT) {
#pragma unroll
        for (int h = 0; h < 8; h++) {
            const int dim = (tid >> 4) + 16 * h, piece = tid & 15, lane = 16 * (piece >> 2) + (dim & 15);
            if (first + 8 * piece >= ld) continue;
            const uint32_t c = *(const uint32_t *)(tile + chunk_of(KV4_V, h, lane) + 4 * (piece & 3));
            *(u32x4 *)(v + (bh * 128 + dim) * ld + first + 8 * piece) =
                decode8(c, scale_of(tile[scale_at(KV4_VS, h, lane)]));  // zeros past P
        }
    } else {
        // four dimensions of eight keys per thread and step: rows of 256 B by 32 threads
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int d4 = tid & 31, oct = (tid >> 5) + 8 * h, g = oct >> 2;
            u32x4 w[4];
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const int dim = 4 * d4 + d, j = dim >> 4, lane = 16 * g + (dim & 15);
                w[d] = decode8(*(const uint32_t *)(tile + chunk_of(KV4_V, j, lane) + 4 * (oct & 3)),
                               scale_of(tile[scale_at(KV4_VS, j, lane)]));
            }
            const int64_t key0 = first + 8 * oct;
#pragma unroll
            for (int n = 0; n < 8; n++) {
                if (key0 + n >= P) break;
                const uint32_t sel = n & 1 ? 0x07060302u : 0x05040100u;
                *(u32x2 *)(v + (bh * P + key0 + n) * 128 + 4 * d4) =
                    u32x2{__builtin_amdgcn_perm(w[1][n >> 1], w[0][n >> 1], sel), __builtin_amdgcn_perm(w[3][n >> 1], w[2][n >> 1], sel)};
            }
        }
    }
}

}  // namespace

int64_t kv4_layer_bytes(int64_t bh, int64_t p) { return bh * ((p + KV4_KEYS - 1) / KV4_KEYS) * KV4_TILE; }

hipError_t launch_store4(const uint16_t *k, const uint16_t *v, int64_t vt_ld, int64_t b, int64_t h, int64_t p,
                         const uint8_t *kvalid, int64_t valid_ld, uint8_t *tiles, float *norm_part, float *norm,
                         hipStream_t stream) {
    const int64_t bh = b * h, T = (p + KV4_KEYS - 1) / KV4_KEYS;
    if (bh <= 0 || p <= 0) return hipSuccess;
    if (bh > 65535 || T >= (int64_t)1 << 24 || (vt_ld && (vt_ld < p || vt_ld % 8))) return hipErrorInvalidValue;
    const int parts = (int)std::min<int64_t>(T * bh, QK_NORM_PARTS);
    store_k4_kernel<<<dim3((unsigned)parts), dim3(256), 0, stream>>>(k, p, h, kvalid, valid_ld, T, T * bh, tiles, norm_part);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (vt_ld)
        store_vt4_kernel<<<dim3((unsigned)T, (unsigned)bh), dim3(256), 0, stream>>>(v, vt_ld, p, h, kvalid, valid_ld, tiles,
                                                                                   norm_part, parts, norm);
    else
        store_v4_kernel<<<dim3((unsigned)((T + 1) / 2), (unsigned)bh), dim3(256), 0, stream>>>(v, p, T, tiles, norm_part,
                                                                                              parts, norm);
    return hipGetLastError();
}

hipError_t launch_load4(const uint8_t *tiles, int64_t bh, int64_t p, int64_t vt_ld, uint16_t *k, uint16_t *v,
                        hipStream_t stream) {
    const int64_t T = (p + KV4_KEYS - 1) / KV4_KEYS;
    if (bh <= 0 || p <= 0) return hipSuccess;
    if (bh > 65535 || T >= (int64_t)1 << 24 || (vt_ld && (vt_ld < p || vt_ld % 8))) return hipErrorInvalidValue;
    const dim3 grid((unsigned)T, (unsigned)bh, 2);
    if (vt_ld)
        load4_kernel<true><<<grid, dim3(256), 0, stream>>>(tiles, p, vt_ld, k, v);
    else
        load4_kernel<false><<<grid, dim3(256), 0, stream>>>(tiles, p, 0, k, v);
    return hipGetLastError();
}

}  // namespace qimm
