// Attention of few queries over a prefix cache held in 4 bits (kv4.h) and own bf16 keys,
// gfx950. Many queries take attention.hip over the expanded layer (attn4_takes).
//
// O = softmax(scale Q [K4 ; K]^T) [V4 ; V], hidden keys at -inf. One pass over the keys
// with the running maximum and sum; f32 scores, sums and output, rounded to bf16 once.
//
// What bounds it: the cache's bytes, 4.25 bits a value, as long as the arithmetic beside
// them stays below: HBM gives a CU about 13 B a clock, 25 values, so a decoding of two VALU
// operations a value would already use up the SIMDs. The matrix pipe takes the codes and
// their powers of two as they lie (v_mfma_scale_f32_16x16x128_f8f6f4, A = keys or values
// in e2m1), so nothing is decoded. The other operand is e4m3 there, four significant bits:
// queries and probabilities go in as the sum of two, x = hi + lo 2^-5, hi = e4m3(x) and
// lo = e4m3((x - hi) 2^5), which holds a bf16 query's eight bits exactly (down to 2^-22
// of its row's largest) and a probability to 2^-9, as the rounding to bf16 of the other
// kernels does. Two products of 128 deep cost the matrix pipe what the bf16 ones would.
//
// A workgroup is 16 queries of one head and a share of the keys, four waves taking
// tiles of 128 keys in turn (64 own keys); a tile's 17 KB go straight into registers, the
// next tile's keys while this one's softmax and P V run, its values after that: nothing
// waits on a barrier until the waves' sums are joined through LDS. With several shares
// (few rows, long caches) a second launch joins them.
#include <algorithm>

#include "kernels.h"
#include "kv4.h"

namespace qimm {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int OWN_KEYS = 64;

__device__ __forceinline__ i32x8 widen(u32x4 c) {
    return i32x8{(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0};
}

// four values below 448 as e4m3 hi (one word) and lo 2^5
__device__ __forceinline__ void split4(float a, float b, float c, float d, int &hi, int &lo) {
    int h = 0;
    h = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, h, false);
    h = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, h, true);
    const f32x2 ab = __builtin_amdgcn_cvt_pk_f32_fp8(h, false), cd = __builtin_amdgcn_cvt_pk_f32_fp8(h, true);
    int l = 0;
    l = __builtin_amdgcn_cvt_pk_fp8_f32((a - ab[0]) * 32.f, (b - ab[1]) * 32.f, l, false);
    l = __builtin_amdgcn_cvt_pk_fp8_f32((c - cd[0]) * 32.f, (d - cd[1]) * 32.f, l, true);
    hi = h;
    lo = l;
}

struct Attn4 {
    const uint16_t *q;      // [B,H,Sq,128]
    const uint8_t *tiles;   // [B*H][T] tiles
    int64_t P, T;
    const uint16_t *k_own;  // [B,H,So,128]
    const uint16_t *vt_own; // [B,H,128,So]
    int64_t So;
    const uint8_t *kvalid;  // [B][P + So] or null
    int64_t H, Sq;
    float sl2;              // softmax scale * log2 e, >= 0 (q's sign is turned with `flip`)
    uint32_t flip;          // 0x80008000 where the scale is negative
    uint16_t *out;          // [B,Sq,H*128]
    float *part;            // shares > 1: O [share][B*H*Sq][128], then (m, l) [share][B*H*Sq]
    int shares;
    uint32_t qtiles;        // tiles of 16 queries
    uint32_t spread;        // heads x shares are a multiple of the XCDs
};

template <bool MASKED>
__global__ __launch_bounds__(256, 2) void attn4_kernel(const Attn4 a) {
    constexpr int PITCH = 132;  // floats per query row in LDS
    __shared__ __attribute__((aligned(16))) float so[4 * 16 * PITCH];
    __shared__ float sm[4][16], sl[4][16];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int l16 = lane & 15, lg = lane >> 4;
    // The query tiles of one share of a head run next to each other on one XCD (workgroups
    // go to the eight in turn), where the second one finds the keys in L2.
    uint32_t at = blockIdx.x, qt;
    if (a.spread) {
        qt = (at >> 3) % a.qtiles;
        at = (at >> 3) / a.qtiles * 8 + (at & 7);
    } else {
        qt = at % a.qtiles;
        at /= a.qtiles;
    }
    const int share = (int)(at % a.shares);
    const int64_t bh = at / a.shares, b = bh / a.H, q0 = (int64_t)qt * 16;
    const int64_t items = a.T + (a.So + OWN_KEYS - 1) / OWN_KEYS;
    const int64_t first = items * share / a.shares, last = items * (share + 1) / a.shares;
    const uint8_t *tiles = a.tiles + bh * a.T * KV4_TILE;

    f32x4 o[8] = {};  // [d tile]: dimensions 16 j + 4 lg + r of query l16
    float m = -INFINITY, l = 0.f;

    u32x4 kc[8], vc[8];
    int ks[2], vs[2];
    auto load_k = [&](int64_t it) __attribute__((always_inline)) {
        const uint8_t *t = tiles + it * KV4_TILE;
#pragma unroll
        for (int i = 0; i < 8; i++) kc[i] = *(const u32x4 *)(t + (i * 64 + lane) * 16);
#pragma unroll
        for (int i = 0; i < 2; i++) ks[i] = *(const int *)(t + KV4_KS + (i * 64 + lane) * 4);
    };
    auto load_v = [&](int64_t it) __attribute__((always_inline)) {
        const uint8_t *t = tiles + it * KV4_TILE + KV4_V;
#pragma unroll
        for (int j = 0; j < 8; j++) vc[j] = *(const u32x4 *)(t + (j * 64 + lane) * 16);
#pragma unroll
        for (int j = 0; j < 2; j++) vs[j] = *(const int *)(t + (KV4_VS - KV4_V) + (j * 64 + lane) * 4);
    };
    // The running maximum over the N scores of a lane's query and its three other lanes',
    // with the sums taken along; the scores become 2^(8 - e) exp(scale (s - max)), hidden ones 0,
    // and e is returned: 0, or of a tile of the cache the power of two of its own largest (from
    // -100 on), so that e4m3, which ends at 2^-23 of the largest with its lo, holds the keys of
    // other tiles than that of a key that takes nearly all. `seen` has a bit per score.
    auto softmax = [&](float *s, auto count, bool some, uint32_t seen) __attribute__((always_inline)) -> int {
        constexpr int N = decltype(count)::value;
        if (some)
#pragma unroll
            for (int e = 0; e < N; e++) s[e] = (seen >> e) & 1u ? s[e] : -INFINITY;
        float mx = s[0];
#pragma unroll
        for (int e = 1; e < N; e++) mx = fmaxf(mx, s[e]);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float top = mx;
        mx = fmaxf(mx, m);
        if (__ballot(mx > m)) {
            // a lane without a visible key so far has sums of 0
            const float al = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mx) * a.sl2);
            m = mx;
            l *= al;
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int r = 0; r < 4; r++) o[j][r] *= al;
        }
        // (no visible key, or all of them infinite: -100, of no consequence)
        const int e2 = N == 32 ? (int)fmaxf(__builtin_ceilf((top - mx) * a.sl2), -100.f) : 0;
        const float c = (float)(8 - e2) - (mx == -INFINITY ? 0.f : mx * a.sl2);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < N; e++) {
            float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], a.sl2, c));
            if (some) p = (seen >> e) & 1u ? p : 0.f;
            s[e] = p;
            sum += p;
        }
        l += __builtin_amdgcn_ldexpf(sum, e2);
        return e2;
    };
    // visible keys of 64 from key k0 of the P + So, the first `have` of them there (have >= 1)
    auto validity = [&](int64_t k0, int have) __attribute__((always_inline)) -> uint64_t {
        bool ok = lane < have;
        if constexpr (MASKED) ok = ok && a.kvalid[b * (a.P + a.So) + k0 + min(lane, have - 1)] != 0;
        return __ballot(ok);
    };
    // the same of tile i's 128 keys in two steps: the bytes, and the masks. A tile without a
    // visible key is neither read nor multiplied.
    struct Bytes {
        uint32_t lo, hi;
    };
    auto bytes_of = [&](int64_t i) __attribute__((always_inline)) -> Bytes {
        if constexpr (!MASKED) return {1, 1};
        const int64_t left = a.P - 1 - i * KV4_KEYS;
        const uint8_t *p = a.kvalid + b * (a.P + a.So) + i * KV4_KEYS;
        return {p[min((int64_t)lane, left)], p[min((int64_t)lane + 64, left)]};
    };
    uint64_t seen_lo = 0, seen_hi = 0;
    auto masks_of = [&](int64_t i, Bytes y) __attribute__((always_inline)) {
        const int have = (int)min(a.P - i * KV4_KEYS, (int64_t)KV4_KEYS);
        seen_lo = __ballot(lane < have && y.lo != 0);
        seen_hi = __ballot(lane + 64 < have && y.hi != 0);
    };

    int64_t it = first + wave;
    const int64_t end = min(last, a.T);
    if (it < end) {
        masks_of(it, bytes_of(it));
        if (seen_lo | seen_hi) {
            load_k(it);
            load_v(it);
        }
    }

    // ---- queries: lane (l16, lg) holds dimensions 16 lg .. + 15 and 64 + 16 lg .. + 15 of query
    // l16, scaled by a power of two so that the row's largest lies in [128, 256) ----
    i32x8 qhi, qlo;
    int qsc;  // scale bytes: hi, lo
    {
        const int64_t qi = min(q0 + l16, a.Sq - 1);
        const u32x4 *src = (const u32x4 *)(a.q + (bh * a.Sq + qi) * 128 + 16 * lg);
        u32x4 w[4];
        uint32_t mag = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            w[e] = src[8 * (e >> 1) + (e & 1)];
#pragma unroll
            for (int x = 0; x < 4; x++) mag = max(mag, max(w[e][x] & 0x7fffu, (w[e][x] >> 16) & 0x7fffu));
        }
        mag = max(mag, (uint32_t)__shfl_xor((int)mag, 16));
        mag = max(mag, (uint32_t)__shfl_xor((int)mag, 32));
        const int ex = (int)(mag >> 7);                            // biased exponent of the row's largest
        const int by = ex == 255 ? 255 : max(ex - 7, 6);           // 2^(ex - 134), biased; no number: NaN
        const float up = __uint_as_float((uint32_t)(254 - min(by, 253)) << 23);
        qsc = by | (by == 255 ? 255 : by - 5) << 8;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t x = w[e >> 1][2 * (e & 1)] ^ a.flip, y = w[e >> 1][2 * (e & 1) + 1] ^ a.flip;
            int hi, lo;
            split4(__uint_as_float(x << 16) * up, __uint_as_float(x & 0xffff0000u) * up, __uint_as_float(y << 16) * up,
                   __uint_as_float(y & 0xffff0000u) * up, hi, lo);
            qhi[e] = hi;
            qlo[e] = lo;
        }
    }

    for (; it < end; it += 4) {
        const int64_t next = it + 4;
        const Bytes ny = next < end ? bytes_of(next) : Bytes{0, 0};
        const bool any = seen_lo | seen_hi, some = (seen_lo & seen_hi) != ~0ull;
        const uint32_t seen = (uint32_t)((seen_lo >> (16 * lg)) & 0xffffu) | (uint32_t)((seen_hi >> (16 * lg)) & 0xffffu) << 16;
        f32x4 acc[8] = {};
        if (any) {
#define QK(i, q, sel) \
    acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(kc[i]), q, acc[i], 4, 0, i & 3, ks[i >> 2], sel, qsc);
            QK(0, qhi, 0) QK(1, qhi, 0) QK(2, qhi, 0) QK(3, qhi, 0) QK(4, qhi, 0) QK(5, qhi, 0) QK(6, qhi, 0) QK(7, qhi, 0)
            QK(0, qlo, 1) QK(1, qlo, 1) QK(2, qlo, 1) QK(3, qlo, 1) QK(4, qlo, 1) QK(5, qlo, 1) QK(6, qlo, 1) QK(7, qlo, 1)
#undef QK
        }
        seen_lo = seen_hi = 0;
        if (next < end) masks_of(next, ny);
        const bool more = seen_lo | seen_hi;
        if (more) load_k(next);
        if (any) {
            float s[32];
#pragma unroll
            for (int e = 0; e < 32; e++) s[e] = acc[e >> 2][e & 3];
            const int e2 = softmax(s, std::integral_constant<int, 32>{}, some, seen);
            i32x8 ph, pl;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                int hi, lo;
                split4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3], hi, lo);
                ph[i] = hi;
                pl[i] = lo;
            }
            const int psc = (127 | 122 << 8) + e2 * 257;  // scale bytes: hi, lo
#define PV(j, p, sel) \
    o[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(vc[j]), p, o[j], 4, 0, j & 3, vs[j >> 2], sel, psc);
            PV(0, ph, 0) PV(1, ph, 0) PV(2, ph, 0) PV(3, ph, 0) PV(4, ph, 0) PV(5, ph, 0) PV(6, ph, 0) PV(7, ph, 0)
            PV(0, pl, 1) PV(1, pl, 1) PV(2, pl, 1) PV(3, pl, 1) PV(4, pl, 1) PV(5, pl, 1) PV(6, pl, 1) PV(7, pl, 1)
#undef PV
        }
        if (more) load_v(next);
    }

    // ---- own keys, 64 at a time in two groups of 32 (bf16 products of 32 deep): row m of
    // product i is key 8 (m / 4) + 4 i + m % 4, so the lane's scores are the eight keys
    // 8 lg .. of its probability operand ----
    for (; it < last; it += 4) {
        const int64_t key0 = (it - a.T) * OWN_KEYS;
        const int have = (int)min(a.So - key0, (int64_t)OWN_KEYS);
        const uint64_t ok = validity(a.P + key0, have);
        const uint16_t *kb = a.k_own + (bh * a.So + key0) * 128;
        const uint16_t *vb = a.vt_own + bh * 128 * a.So + key0;
        const bool some = ok != ~0ull;
        const uint32_t seen = (uint32_t)((ok >> (8 * lg)) & 0xffu) | (uint32_t)((ok >> (32 + 8 * lg)) & 0xffu) << 8;
        // the loads of the keys and half of the values together, then the other half
        bf16x8 qf[4], kq[2][2][4];
        u32x4 vq[2][8];
        const uint16_t *qp = a.q + (bh * a.Sq + min(q0 + l16, a.Sq - 1)) * 128 + 8 * lg;
#pragma unroll
        for (int e = 0; e < 4; e++) qf[e] = __builtin_bit_cast(bf16x8, *(const u32x4 *)(qp + 32 * e) ^ a.flip);
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint16_t *kp = kb + (int64_t)min(32 * g + 8 * (l16 >> 2) + 4 * i + (l16 & 3), have - 1) * 128 + 8 * lg;
#pragma unroll
                for (int e = 0; e < 4; e++) kq[g][i][e] = *(const bf16x8 *)(kp + 32 * e);
            }
        auto load_vq = [&](int g) __attribute__((always_inline)) {
            const int k8 = 32 * g + 8 * lg;  // the lane's eight keys
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint16_t *row = vb + (int64_t)(16 * j + l16) * a.So;  // from key0 on
                if (have == OWN_KEYS) {
                    __builtin_memcpy(&vq[g][j], row + k8, 16);  // at any alignment
                } else if (32 * g >= have) {
                    vq[g][j] = u32x4{};
                } else if (a.So >= 8) {
                    // the row's last eight keys, shifted down to the lane's, zeros after them
                    const int from = min(k8, have - 8), drop = min(k8 - from, 8);
                    uint64_t v[2];
                    __builtin_memcpy(v, row + from, 16);
                    const int d = 16 * (drop & 3);
                    const uint64_t lo = drop & 4 ? v[1] : v[0], hi = drop & 4 ? 0 : v[1];
                    v[0] = drop == 8 ? 0 : d ? lo >> d | hi << (64 - d) : lo;
                    v[1] = drop == 8 ? 0 : hi >> d;
                    __builtin_memcpy(&vq[g][j], v, 16);
                } else {  // fewer than eight in all: the first lanes'
                    vq[g][j] = u32x4{};
#pragma unroll
                    for (int e = 0; e < 7; e++)
                        if (e < have && lg == 0) vq[g][j][e >> 1] |= (uint32_t)row[e] << (16 * (e & 1));
                }
            }
        };
        load_vq(0);
        float s[16];
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 4; e++) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kq[g][i][e], qf[e], acc, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; r++) s[8 * g + 4 * i + r] = acc[r];
            }
        load_vq(1);
        softmax(s, std::integral_constant<int, 16>{}, some, seen);
#pragma unroll
        for (int g = 0; g < 2; g++) {
            const u32x4 p = u32x4{pack_bf16x2(s[8 * g], s[8 * g + 1]), pack_bf16x2(s[8 * g + 2], s[8 * g + 3]),
                                  pack_bf16x2(s[8 * g + 4], s[8 * g + 5]), pack_bf16x2(s[8 * g + 6], s[8 * g + 7])};
            const uint32_t keep = (seen >> (8 * g)) & 0xffu;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if (some)  // what a hidden key holds does not count, a NaN either
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        vq[g][j][e] &= ((keep >> (2 * e)) & 1u ? 0xffffu : 0u) | ((keep >> (2 * e + 1)) & 1u ? 0xffff0000u : 0u);
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, vq[g][j]), __builtin_bit_cast(bf16x8, p),
                                                               o[j], 0, 0, 0);
            }
        }
    }

    // ---- the four waves' sums ----
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (lg == 0) {
        sm[wave][l16] = m;
        sl[wave][l16] = l;
    }
    float *mine = so + (wave * 16 + l16) * PITCH + 4 * lg;
#pragma unroll
    for (int j = 0; j < 8; j++) *(f32x4 *)(mine + 16 * j) = o[j];
    __syncthreads();
    constexpr int TPQ = 16, DPT = 8;  // threads per query, dimensions per thread
    const int ql = tid / TPQ, d0 = (tid % TPQ) * 4;
    const int64_t qi = q0 + ql;
    if (qi >= a.Sq) return;
    float mm = fmaxf(fmaxf(sm[0][ql], sm[1][ql]), fmaxf(sm[2][ql], sm[3][ql])), ll = 0.f, f[4];
#pragma unroll
    for (int w = 0; w < 4; w++) {
        f[w] = sm[w][ql] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((sm[w][ql] - mm) * a.sl2);
        ll += sl[w][ql] * f[w];
    }
    const int64_t row = bh * a.Sq + qi, rows = (int64_t)(gridDim.x / (a.qtiles * (uint32_t)a.shares)) * a.Sq;
    if (a.shares > 1 && tid % TPQ == 0) {
        float *ml = a.part + (int64_t)a.shares * rows * 128 + ((int64_t)share * rows + row) * 2;
        ml[0] = mm;
        ml[1] = ll;
    }
    const float inv = 1.0f / ll;  // a query that sees no key: 0 / 0, as the softmax of -inf
#pragma unroll
    for (int e = 0; e < DPT / 4; e++) {
        const int d = d0 + 4 * TPQ * e;
        f32x4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const f32x4 x = *(const f32x4 *)(so + (w * 16 + ql) * PITCH + d);
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] += x[r] * f[w];
        }
        if (a.shares > 1)
            *(f32x4 *)(a.part + ((int64_t)share * rows + row) * 128 + d) = v;
        else
            *(u32x2 *)(a.out + ((b * a.Sq + qi) * a.H + bh % a.H) * 128 + d) =
                u32x2{pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv)};
    }
}

// Joins the shares of a row, one wave per row, two dimensions per lane.
__global__ __launch_bounds__(256) void attn4_join_kernel(const float *__restrict__ part, int shares, int64_t rows, int64_t H,
                                                         int64_t Sq, float sl2, uint16_t *__restrict__ out) {
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const int lane = threadIdx.x & 63;
    const f32x2 *ml = (const f32x2 *)(part + (int64_t)shares * rows * 128);
    // lane s has share s's maximum and sum (at most 64 shares)
    const f32x2 mine = lane < shares ? ml[lane * rows + row] : f32x2{-INFINITY, 0.f};
    float mm = mine[0];
    for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o));
    const float f = mine[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mine[0] - mm) * sl2);
    const float ll = wave_sum(mine[1] * f);
    f32x2 v{0.f, 0.f};
    for (int s = 0; s < shares; s++) {
        const f32x2 x = *(const f32x2 *)(part + ((int64_t)s * rows + row) * 128 + 2 * lane);
        const float fs = __shfl(f, s);
        v[0] += x[0] * fs;
        v[1] += x[1] * fs;
    }
    const float inv = 1.0f / ll;
    const int64_t bh = row / Sq, qi = row % Sq;
    *(uint32_t *)(out + ((bh / H * Sq + qi) * H + bh % H) * 128 + 2 * lane) = pack_bf16x2(v[0] * inv, v[1] * inv);
}

// Shares of the keys: two workgroups per CU, each share at least a tile for every wave, at most 64;
// one up to four tiles a wave, which cost less than the joining launch (32 heads, one query: 1500
// keys 13.9 us in shares, 10.7 in one; 2040 keys 13.9 and 12.3).
int shares_of(int64_t wgs, int64_t items) {
    if (items <= 16) return 1;
    const int64_t want = 2 * (int64_t)std::max(device_cu_count(), 1);
    return (int)std::max<int64_t>(1, std::min<int64_t>({want / wgs, (items + 3) / 4, 64}));
}

}  // namespace

// more than one share only with at most two workgroups of 16 rows per CU
size_t attn4_scratch_bytes() { return (size_t)std::max(device_cu_count(), 1) * 2 * 16 * (128 + 2) * 4; }

// Which calls this kernel takes: those it is estimated to do before the expansion of the layer
// and attention.hip, in us. Here 16 queries over 128 keys of the cache take 1.39 ns with the
// card full, over 64 own keys 2.7 ns (8 requests of 32 heads, 4299 keys: 256 queries 194 and
// with as many own keys 231, 1024 queries 787 and 1469). There the expansion moves 2.53 B a
// value at 5 TB/s and two launches take about 12; a round of 256-query tiles takes 2.15 per 64
// keys (masked 1.8 and no half tiles) and 8, 0.63 of that where half tiles fill at most one
// per CU. Measured, here / there: 1 x 32 heads over 333 keys, 64 queries 7 / 20, 512 with as
// many own 39 / 31; over 4299, 512 with as many own 74 / 121, 1024 190 / 132 and without own
// keys 99 / 122; 8 x 32 heads over 4299 with as many own, 256 231 / 332, 512 560 / 461.
bool attn4_takes(int64_t bh, int64_t sq, int64_t p, int64_t so, bool masked) {
    const double cus = (double)std::max(device_cu_count(), 1), part = 256.0 / cus;
    const double tiles = (double)bh * (double)((sq + 15) / 16);
    if (tiles >= (double)(1 << 24)) return false;  // 2^32 threads
    const double here = 8.0 + part * tiles * (1.39e-3 * (double)((p + KV4_KEYS - 1) / KV4_KEYS) +
                                              2.7e-3 * (double)((so + OWN_KEYS - 1) / OWN_KEYS));
    const double blocks = (double)((p + 63) / 64 + (so + 63) / 64), n8 = (double)((sq + 255) / 256 * bh);
    const bool half = !masked && (double)((sq + 127) / 128 * bh) <= cus;
    const double rounds = half ? 0.63 : (double)(int64_t)((n8 + cus - 1) / cus);
    const double there = 12.0 + (double)bh * (double)p * 256.0 * 2.53 / 5e6 + rounds * ((masked ? 1.8 : 2.15) * blocks + 8.0);
    return here <= there;
}

hipError_t launch_attn4(const uint16_t *q, const uint8_t *tiles, int64_t p, const uint16_t *k_own, const uint16_t *vt_own,
                        int64_t so, const uint8_t *kvalid, int64_t b, int64_t h, int64_t sq, float scale, float *scratch,
                        uint16_t *out, hipStream_t stream) {
    if (sq <= 0 || b <= 0 || h <= 0) return hipSuccess;
    if (p < 0 || so < 0 || p + so <= 0 || !scratch) return hipErrorInvalidValue;
    const int64_t bh = b * h, T = (p + KV4_KEYS - 1) / KV4_KEYS, items = T + (so + OWN_KEYS - 1) / OWN_KEYS;
    const int64_t qt = (sq + 15) / 16;
    const int shares = shares_of(bh * qt, items);
    if (bh * qt * shares >= (int64_t)1 << 24) return hipErrorInvalidValue;
    const float sl2 = scale * 1.4426950408889634f;
    const Attn4 a{q, tiles, p, T, k_own, vt_own, so, kvalid, h, sq, sl2 < 0.f ? -sl2 : sl2,
                  sl2 < 0.f ? 0x80008000u : 0u, out, scratch, shares, (uint32_t)qt, (uint32_t)(bh * shares % 8 == 0)};
    const dim3 grid((unsigned)(bh * qt * shares));
    if (kvalid)
        attn4_kernel<true><<<grid, dim3(256), 0, stream>>>(a);
    else
        attn4_kernel<false><<<grid, dim3(256), 0, stream>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || shares == 1) return e;
    attn4_join_kernel<<<dim3((unsigned)((bh * sq + 3) / 4)), dim3(256), 0, stream>>>(scratch, shares, bh * sq, h, sq, a.sl2, out);
    return hipGetLastError();
}

}  // namespace qimm
