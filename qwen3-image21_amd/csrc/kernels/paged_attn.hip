// Attention over the paged K/V cache (paged.h), gfx950: the rows of a step, any number per request,
// over their requests' pages.
//
// O = softmax(scale Q K^T) V. Row i of a request's n, of which `len` tokens are in the cache, stands at
// p = len - n + i and sees the keys j <= p (causal) or j < len; in a window of W only j > p - W, and
// j < sinks. One pass over the keys with the running maximum and sum; f32 scores, sums and output,
// rounded to bf16 once; probabilities are rounded to bf16 (2^-8 at most) as the operand of P V.
//
// The query heads of one key head share its keys: a pair is a row and a head of the group, a tile the
// pairs of a request and key head in row order. A wave has 32 of them: it computes S^T = K Q^T with
// v_mfma_f32_32x32x16_bf16, so a lane owns one pair and its maximum and sum need one lane more, and
// O^T += V^T P^T from the registers that S^T leaves.
//
// Few pairs (few_pairs: up to 32, single tokens) are bound by the cache's bytes: HBM gives a CU about 9 B a
// clock, 16 KB of a 32-key tile of 128 dims take it 1900 clocks, its 16 matrix instructions a SIMD 512 and
// the softmax about as many, so the columns of a tile that are empty cost nothing. Four waves take
// tiles of 32 keys in turn straight into registers (two operands of 8 KB in flight each: no LDS, no barrier) and
// join their sums through LDS. One token over 131001 keys of 8 heads: 103 us, 5.2 TB/s.
//
// More (many_pairs) are bound by the matrix pipe and the softmax beside it: four waves share 64-key tiles in
// LDS, where each key is read by 128 pairs. A prompt of 8395 tokens, 32 heads over 8, causal: 585 us, 0.99
// PFLOP/s (two such workgroups on a CU take 2.1 us a tile each, one alone 1.7).
//
// Long requests in few workgroups are split over their keys. The host does not know the lengths, so
// every workgroup counts the rounds of keys of all requests, which gives the rounds of a share and with that
// which share of which request it is itself (piece_of). The shares' sums go through memory; the last ones
// to arrive join them, in a fixed order.
#include <algorithm>
#include <type_traits>

#include "device_common.h"
#include "paged.h"

namespace qimm {
namespace {

// The two forms: pairs of a tile, keys of a round, and the shares: at least GRAIN rounds each, at most MOST of
// a tile, SLOTS in all; `want` workgroups are the aim (Attn), ON_CU a CU.
struct Few {
    static constexpr bool ROWS = false;
    static constexpr int TM = 32, ROUND = 128, GRAIN = 4, MOST = 128, SLOTS = 1280, ON_CU = 4;
};
struct Rows {
    static constexpr bool ROWS = true;
    static constexpr int TM = 128, ROUND = 64, GRAIN = 8, MOST = 64, SLOTS = 640, ON_CU = 2;
};
constexpr int KT = 32;          // keys of a wave's tile, few pairs
// The maximum of a pair whose scores are all -infinity, where that of one that sees no key is -infinity: its
// sum is 0 too, but it gives NaN and not zeros.
constexpr float LOWEST = -3.402823466e38f;
constexpr int FEW_PAIRS = 32;   // more pairs of a request and key head are rows
static_assert(2 * (Few::SLOTS + Rows::SLOTS) * 4 <= PAGED_COUNTER_BYTES, "two counters per slot");

struct Attn {
    const uint16_t *q;
    int64_t q_row, q_head;
    const uint8_t *cache;  // the layer
    int64_t pages;
    const int32_t *tables;
    int64_t max_pages;
    const int32_t *lengths, *starts;
    int32_t R, T;          // requests, rows
    int32_t Hkv, G;        // key heads, query heads of each
    int32_t ps16;          // granules of a page
    uint32_t ps16_magic;   // ceil(2^32 / ps16): x / ps16 = x magic >> 32 for x < 2^27, ps16 <= 32
    int32_t cap;           // keys that a table row has room for
    int32_t causal, window, sinks;  // window 0: none
    float sl2;             // scale * log2 e
    uint16_t *out;
    uint32_t *count;       // arrivals per slot, the few's and the rows', of shares and of teams, zero between
                           // calls; null: no request is long enough to be split
    float *part;           // per slot O [TM][D], then (m, l) [TM]
    int32_t row_pieces;    // workgroups for rows; the others are for few
    int32_t turn;          // of which so many take turns, a multiple of the XCDs
    uint64_t g_magic;      // floor(2^64 / G) + 1: f / G = f g_magic >> 64 for f < 2^32, G > 1
    int32_t want[2];       // workgroups that few pairs, rows are divided into, where they are long enough: four a CU
                           // of few (two fit; the second pair evens out the first), two of rows
};

// pair f's row
__device__ __forceinline__ int row_of_pair(const Attn &a, int f) {
    const uint64_t lo = (uint64_t)(uint32_t)f * (uint32_t)a.g_magic >> 32;
    const int x = (int)(((uint64_t)(uint32_t)f * (uint32_t)(a.g_magic >> 32) + lo) >> 32);
    return a.G == 1 ? f : x;
}

// a request's rows and tokens
struct Req {
    int start, n, len;
};
__device__ __forceinline__ Req req_of(const Attn &a, int r) {
    const int s = a.starts ? min(max(a.starts[r], 0), a.T) : r;
    const int e = a.starts ? min(max(a.starts[r + 1], s), a.T) : min(r + 1, a.T);
    return {s, e - s, min(max(a.lengths[r], 0), a.cap)};
}

// The keys that some pair of `pairs` from `first` on sees: [0, sk) and lo .. hi - 1, as tiles of KEYS: ns of
// the first ones, then from w0 on; pos0, pos1: the positions of the first and last row (-1 before token 0).
struct Range {
    int pos0, pos1, lo, hi, sk, ns, w0, tiles;
};
template <int KEYS>
__device__ __forceinline__ Range range_of(const Attn &a, const Req &q, int first, int pairs) {
    Range g;
    const int i0 = min(row_of_pair(a, first), q.n - 1), i1 = min(q.n - 1, row_of_pair(a, first + pairs - 1));
    g.pos0 = max(a.causal ? q.len - q.n + i0 : q.len - 1, -1);
    g.pos1 = max(a.causal ? q.len - q.n + i1 : q.len - 1, -1);
    g.hi = g.pos1 + 1;
    g.lo = a.window ? max(g.pos0 - a.window + 1, 0) : 0;
    g.sk = a.window ? min(a.sinks, g.hi) : 0;
    g.ns = (g.sk + KEYS - 1) / KEYS;
    g.w0 = g.lo / KEYS;
    if (g.w0 <= g.ns) g.ns = g.w0 = 0;
    g.tiles = g.ns + (g.hi + KEYS - 1) / KEYS - g.w0;
    return g;
}
__device__ __forceinline__ int tile_at(const Range &g, int v) { return v < g.ns ? v : v - g.ns + g.w0; }

// The maximum m of a lane's pair after tiles first, first + STEP, ... of KEYS: LOWEST where it is -infinity and
// the pair sees a key of them all the same. Behind the loops: asked of every tile there, it took 2% of a prompt
// in a window. Out of the way of waves that have nothing to look for (333 keys of 32 heads 6.74 us inline, 6.65).
template <int KEYS, int STEP>
__device__ __forceinline__ float lowest_of(const Attn &a, const int32_t *table, const Range &g, int first, int last, float m, int pos, int low, int sk) {
    bool asks = m == -INFINITY && pos >= 0 && first < last;
    if (__builtin_expect(__ballot(asks) == 0, 1)) return m;
    if (asks) {
        const int from = tile_at(g, first) * KEYS;
        asks = from <= pos && (from < sk || tile_at(g, last - 1) * KEYS + KEYS - 1 > low);
    }
#pragma unroll 1
    for (int v = first; __ballot(asks) && v < last; v += STEP) {
#pragma unroll 1
        for (int i = 0; i < KEYS / 16; i++) {
            const uint32_t x = tile_at(g, v) * (KEYS / 16) + i, k = __umulhi(x, a.ps16_magic) + (a.ps16 == 1 ? x : 0);
            const int page = (int64_t)k < a.max_pages ? table[k] : -1, key = (int)x * 16;
            if (asks && page >= 0 && page < a.pages && key <= pos && (key + 15 > low || key < sk)) {  // (low < pos)
                m = LOWEST;
                asks = false;
            }
        }
    }
    return m;
}

// A request's tiles of the form's, and the rounds of the keys that any of them sees, at most.
template <typename F>
__device__ __forceinline__ int tiles_of(const Attn &a, const Req &q) {
    const int pairs = q.n * a.G;
    return (pairs > FEW_PAIRS) == F::ROWS ? (pairs + F::TM - 1) / F::TM : 0;
}
template <typename F>
__device__ __forceinline__ int rounds_of(const Attn &a, const Req &q) {
    int64_t keys = q.len;
    if (a.window) keys = min(keys, (int64_t)a.sinks + a.window + F::TM / a.G + 2 * F::ROUND);
    return (int)((keys + F::ROUND - 1) / F::ROUND);
}

// What a workgroup takes: share `share` of `shares` of tile `tile` of request r's pairs for key head h; slot:
// the tile's first of the shares' slots. rq: the request.
struct Piece {
    int r, h, tile, share, shares, slot;
    Req rq;
};

// sums over 256 threads: those before this one
__device__ __forceinline__ int64_t scan256(int64_t v, int64_t *part, int64_t &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t x = __shfl_up(s, o);
        if (lane >= o) s += x;
    }
    __syncthreads();
    if (lane == 63) part[wave] = s;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        if (w < wave) before += part[w];
        total += part[w];
    }
    return before + s - v;
}

// A request's tiles and shares with `chunk` rounds a share (0: nothing is split), its pieces and, of a split
// one, their slots.
struct Split {
    int tiles, shares, pieces, slots;
};
template <typename F>
__device__ __forceinline__ Split split_of(const Attn &a, const Req &q, int chunk) {
    Split s;
    s.tiles = tiles_of<F>(a, q);
    s.shares = 1;
    const int rounds = rounds_of<F>(a, q);
    if (chunk && s.tiles && rounds > F::GRAIN) s.shares = max(min((rounds + chunk - 1) / chunk, F::MOST), 1);
    s.pieces = (int)min((int64_t)s.tiles * s.shares * a.Hkv, (int64_t)1 << 24);
    s.slots = s.shares > 1 ? s.pieces : 0;
    return s;
}
// Rounds of a share, of `rounds` of all tiles for one head and `tiles` of them, and whether so many pieces and
// slots of it will do (else a little longer shares are tried, at the end nothing is split). Rows that one round of
// workgroups takes are divided into no more than that, those of not much more than one into shares half as
// long: 136 tiles of 100 rounds in 544 shares took 139 us, in 408 112 (with their join as it was then). Shares may
// be of half a GRAIN as long as each has a CU of its own: one token over 4000 keys of 8 heads 14.5 us in 64
// shares, 11.7 in 128, but 8 of them over 2000 18.4 in 256 and 19.5 in 512; 221 rows of 3 heads over 10114 keys of
// one 41.0 in 120 shares, 32.7 in 240 (with smaller teams of the join). Requests of up to a GRAIN are not split: 333 keys of 32 heads took 8.4 us whole (6.6 since) and 10.2 in two shares.
template <typename F>
__device__ __forceinline__ int chunk_of(const Attn &a, float rounds, int64_t tiles) {
    const int want = a.want[F::ROWS], c = (int)(rounds * (float)a.Hkv / (float)want) + 1;
    const int least = rounds * (float)a.Hkv <= (float)(want / F::ON_CU * (F::GRAIN / 2)) ? F::GRAIN / 2 : F::GRAIN;
    return max(least, F::ROWS && tiles * a.Hkv > want && tiles * a.Hkv < 2 * want ? (c + 1) / 2 : c);
}
template <typename F>
__device__ __forceinline__ bool will_do(const Attn &a, int64_t pieces, int64_t slots, int64_t tiles, int most) {
    if (slots == 0) return true;
    return slots <= F::SLOTS && pieces <= most && !(F::ROWS && tiles * a.Hkv <= a.want[1] && pieces > a.want[1]);
}
// Piece `i` of a request: heads fastest, the last tiles first (under causal rows
// they see the most keys).
template <typename F>
__device__ __forceinline__ Piece piece_in(const Attn &a, int r, const Req &q, const Split &s, int i, int slots_before) {
    Piece p;
    const int x = i / a.Hkv;
    p.r = r;
    p.h = i - x * a.Hkv;
    p.tile = s.tiles - 1 - x / s.shares;
    p.share = x % s.shares;
    p.shares = s.shares;
    p.slot = (F::ROWS ? Few::SLOTS : 0) + slots_before + (p.tile * a.Hkv + p.h) * s.shares;
    p.rq = q;
    return p;
}
// sums over the lanes up to this one
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
    const auto from = [](T x, auto ctrl, auto rows) __attribute__((always_inline)) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value,
                                                                 decltype(rows)::value, 0xf, false));
    };
    v += from(v, std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});  // row_shr 1, 2, 4, 8
    v += from(v, std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
    v += from(v, std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
    v += from(v, std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
    v += from(v, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // row_bcast 15, 31
    v += from(v, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
    return v;
}
template <typename T>
__device__ __forceinline__ T lane_of(T v, int lane) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// The piece of workgroup `item` of at most `most`, in request order; false: there is none. Up to 64
// requests every wave counts them by itself, a lane each; of more, every thread counts its share and the one whose
// share has the piece looks which: as much work as requests times workgroups. A token of each of 2048 requests of 100
// to 2000 keys of 8 heads 988 us, their bytes 1033; but 16384 of up to 520 keys 12 ms, their bytes 0.6.
template <typename F>
__device__ __forceinline__ bool piece_of(const Attn &a, int item, int most, Piece &out) {
    if (!F::ROWS && !a.starts && !a.count) {
        // one tile of every request and key head
        const int r = item / a.Hkv;
        if (r >= a.R) return false;
        out = {r, item - r * a.Hkv, 0, 0, 1, 0, req_of(a, r)};
        return true;
    }
    if (a.R <= 64) {
        const int lane = threadIdx.x & 63;
        Req q = lane < a.R ? req_of(a, lane) : Req{0, 0, 0};
        int chunk = 0, tiles = 0, r = lane;
        if (a.count) {
            const int t = tiles_of<F>(a, q);
            tiles = lane_of(wave_scan(t), 63);
            chunk = chunk_of<F>(a, lane_of(wave_scan((float)t * (float)rounds_of<F>(a, q)), 63), tiles);
        }
        Split s;
        for (;; chunk += (chunk + 7) / 8) {
            s = split_of<F>(a, q, chunk);
            if (!chunk || will_do<F>(a, lane_of(wave_scan(s.pieces), 63), lane_of(wave_scan(s.slots), 63), tiles, most)) break;
        }
        if (F::ROWS && a.R > 1) {
            // the longest shares first: lane i takes the request of rank i
            const int w = s.tiles ? (rounds_of<F>(a, q) + s.shares - 1) / s.shares : -1;
            int rank = 0;
            for (int i = 0; i < a.R; i++) {
                const int x = __builtin_amdgcn_readlane(w, i);
                rank += x > w || (x == w && i < lane);
            }
            rank = (lane < a.R ? rank : lane) * 4;
            q.start = __builtin_amdgcn_ds_permute(rank, q.start);
            q.n = __builtin_amdgcn_ds_permute(rank, q.n);
            q.len = __builtin_amdgcn_ds_permute(rank, q.len);
            r = __builtin_amdgcn_ds_permute(rank, lane);
            s = split_of<F>(a, q, chunk);
        }
        const int pieces = wave_scan(s.pieces), slots = wave_scan(s.slots);
        const uint64_t behind = __ballot(pieces > item);
        if (!behind) return false;
        const int at = __builtin_ctzll(behind);
        const Split mine{lane_of(s.tiles, at), lane_of(s.shares, at), 0, 0};
        out = piece_in<F>(a, lane_of(r, at), Req{lane_of(q.start, at), lane_of(q.n, at), lane_of(q.len, at)}, mine,
                          item - lane_of(pieces - s.pieces, at), lane_of(slots - s.slots, at));
        return true;
    }
    __shared__ int64_t part[4];
    __shared__ Piece found;
    const int c = (a.R + 255) / 256, r0 = min((int)threadIdx.x * c, a.R), r1 = min(r0 + c, a.R);
    int chunk = 0;
    int64_t tiles = 0, all, slots_all;
    if (a.count) {
        int64_t t = 0, rounds = 0;
        for (int r = r0; r < r1; r++) {
            const Req q = req_of(a, r);
            const int n = tiles_of<F>(a, q);
            t += n;
            rounds += (int64_t)n * rounds_of<F>(a, q);
        }
        scan256(t, part, tiles);
        scan256(rounds, part, all);
        chunk = chunk_of<F>(a, (float)all, tiles);
    }
    int64_t mine, at, slots_mine, slots_at;
    for (;; chunk += (chunk + 7) / 8) {
        mine = slots_mine = 0;
        for (int r = r0; r < r1; r++) {
            const Split s = split_of<F>(a, req_of(a, r), chunk);
            mine += s.pieces;
            slots_mine += s.slots;
        }
        at = scan256(mine, part, all);
        slots_at = scan256(slots_mine, part, slots_all);
        if (!chunk || will_do<F>(a, all, slots_all, tiles, most)) break;
    }
    if (item >= all) return false;
    if (item >= at && item < at + mine)
        for (int r = r0;; r++) {
            const Req q = req_of(a, r);
            const Split s = split_of<F>(a, q, chunk);
            if (item < at + s.pieces) {
                found = piece_in<F>(a, r, q, s, (int)(item - at), (int)slots_at);
                break;
            }
            at += s.pieces;
            slots_at += s.slots;
        }
    __syncthreads();
    const int *src = (const int *)&found;
    int *dst = (int *)&out;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Piece) / 4); i++) dst[i] = __builtin_amdgcn_readfirstlane(src[i]);
    return true;
}

// the larger magnitudes of two pairs of bf16 values, as bits
__device__ __forceinline__ uint32_t magnitude2(uint32_t m, uint32_t w) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
}
// (of values or their magnitudes)
__device__ __forceinline__ bool not_finite2(uint32_t w) {
    return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// The shares' sums cross the XCDs: stored through to and loaded from memory (sc0 sc1), so that a
// share's are there once its stores are done, without a fence that writes back all of an L2.
struct Part {
    __amdgpu_buffer_rsrc_t r;
    static constexpr int SYS = 1 | 16;
    __device__ __forceinline__ Part(const float *base, uint32_t floats)
        : r(__builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)(floats * 4), 0x00020000)) {}
    __device__ __forceinline__ void put4(uint32_t i, f32x4 v) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, i * 4u, 0, SYS);
    }
    __device__ __forceinline__ f32x4 get4(uint32_t i) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, i * 4u, 0, SYS));
    }
    __device__ __forceinline__ void put2(uint32_t i, float x, float y) const {
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(x), __float_as_uint(y)}, r, i * 4u, 0, SYS);
    }
    __device__ __forceinline__ u32x2 get2(uint32_t i) const {
        return __builtin_amdgcn_raw_buffer_load_b64(r, i * 4u, 0, SYS);
    }
};
// floats of a slot, and where slot `slot` starts
template <typename F, int D>
__device__ __forceinline__ constexpr uint32_t slot_floats() {
    return F::TM * (D + 2);
}
template <typename F, int D>
__device__ __forceinline__ const float *slot_at(const Attn &a, int slot) {
    const int64_t few = (int64_t)Few::SLOTS * slot_floats<Few, D>();
    return F::ROWS ? a.part + few + (int64_t)(slot - Few::SLOTS) * slot_floats<F, D>() : a.part + (int64_t)slot * slot_floats<F, D>();
}

// Where a thread's vectors of four sums lie in a slot, i < TM D / 1024 of them a thread: rows of D for few pairs,
// for rows as the waves hold them (a wave's stores are 1 KB in a row).
template <typename F, int D>
__device__ __forceinline__ void vector_at(int i, uint32_t &at, int &pair, int &dim) {
    const int tid = threadIdx.x, lane = tid & 63;
    if (F::ROWS) {
        at = (uint32_t)(tid >> 6) * (32 * D) + i * 256 + lane * 4;
        pair = (tid >> 6) * 32 + (lane & 31);
        dim = 8 * i + 4 * (lane >> 5);
    } else {
        at = (uint32_t)(tid + 256 * i) * 4;
        pair = (tid + 256 * i) / (D / 4);
        dim = at % D;
    }
}

// Joins the sums in n (up to TEAM) slots, `stride` apart from `first` on, by 256 threads: into the output, row(p)
// that of pair p, or into the first of them. fac: TEAM * TM floats of LDS.
constexpr int TEAM = 16;
template <typename F, int D, int I0, int NV, int AT, typename Row>
__device__ __forceinline__ void join_vectors(const Part &pb, int n, uint32_t step, int pairs, const float *fac, bool last, Row row) {
    f32x4 x[NV] = {};
    for (int s0 = 0; s0 < n; s0 += AT) {
        f32x4 y[AT][NV];
#pragma unroll
        for (int s = 0; s < AT; s++)
#pragma unroll
            for (int i = 0; i < NV; i++) {
                uint32_t at;
                int p, d;
                vector_at<F, D>(I0 + i, at, p, d);
                y[s][i] = pb.get4((uint32_t)min(s0 + s, n - 1) * step + at);
            }
#pragma unroll
        for (int s = 0; s < AT; s++)
#pragma unroll
            for (int i = 0; i < NV; i++) {
                uint32_t at;
                int p, d;
                vector_at<F, D>(I0 + i, at, p, d);
                if (s0 + s >= n) continue;  // (read once more)
                // a share that weighs nothing counts too: what it has seen may be no number
                const float f = p < pairs ? fac[(s0 + s) * F::TM + p] : 0.f;
#pragma unroll
                for (int e = 0; e < 4; e++) x[i][e] += y[s][i][e] * f;
            }
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
        uint32_t at;
        int p, d;
        vector_at<F, D>(I0 + i, at, p, d);
        if (p >= pairs) continue;
        if (last)
            *(u32x2 *)(row(p) + d) = u32x2{pack_bf16x2(x[i][0], x[i][1]), pack_bf16x2(x[i][2], x[i][3])};
        else
            pb.put4(at, x[i]);
    }
}
template <typename F, int D, typename Row>
__device__ __forceinline__ void join_shares(const Attn &a, int first, int n, int stride, int pairs, float *fac, bool last, Row row) {
    const uint32_t step = (uint32_t)stride * slot_floats<F, D>();
    const Part pb(slot_at<F, D>(a, first), (uint32_t)(n - 1) * step + slot_floats<F, D>());
    // a share's factor for each pair: exp2 of its maximum relative to the largest, over the sum at last
    const int p = threadIdx.x;
    if (p < pairs) {
        float m[TEAM], mm = -INFINITY, ll = 0.f;
        u32x2 ml[TEAM];
#pragma unroll
        for (int s = 0; s < TEAM; s++) ml[s] = pb.get2((uint32_t)min(s, n - 1) * step + F::TM * D + 2 * p);
#pragma unroll
        for (int s = 0; s < TEAM; s++) {
            m[s] = s < n ? __uint_as_float(ml[s][0]) : -INFINITY;
            mm = fmaxf(mm, m[s]);
        }
#pragma unroll
        for (int s = 0; s < TEAM; s++) {
            m[s] = m[s] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m[s] - mm) * a.sl2);
            ll += __uint_as_float(ml[s][1]) * m[s];
        }
        const float inv = !last ? 1.f : mm == -INFINITY ? 0.f : 1.0f / ll;
#pragma unroll
        for (int s = 0; s < TEAM; s++) fac[s * F::TM + p] = m[s] * inv;
        if (!last) pb.put2(F::TM * D + 2 * p, mm, ll);
    }
    __syncthreads();
    if constexpr (!F::ROWS) {
        if (pairs * (D / 4) <= 256)
            join_vectors<F, D, 0, 1, TEAM>(pb, n, step, pairs, fac, last, row);
        else
            join_vectors<F, D, 0, D / 32, 4>(pb, n, step, pairs, fac, last, row);
    } else {
        // (two shares in flight: with three, teams of 4 read two for nothing, 28.8 us for 27.0 below)
        join_vectors<F, D, 0, D / 16, 2>(pb, n, step, pairs, fac, last, row);
        join_vectors<F, D, D / 16, D / 16, 2>(pb, n, step, pairs, fac, last, row);
    }
}

// Whether the workgroup, whose sums are stored, is the last of n to arrive at a counter, which it leaves zero.
__device__ __forceinline__ bool last_of(uint32_t *counter, int n) {
    __shared__ uint32_t arrived;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        arrived = atomicAdd(counter, 1u);
        if (arrived == (uint32_t)n - 1) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return arrived == (uint32_t)n - 1;
}
// A share's sums are stored: the last of every team of shares joins them, the last of the teams those. A slot of rows
// is 66 KB at D = 128, so their teams are small and join at the same time: 16 rows of 32 heads over 8000 keys
// 34.5 us in teams of 16, 30.5 of 8, 28.5 of 4 (27.0 with two shares read at a time).
template <typename F, int D, typename Row>
__device__ __forceinline__ void arrive(const Attn &a, const Piece &pc, int pairs, float *lds, Row row) {
    constexpr int OF = F::ROWS ? 4 : TEAM;
    static_assert(F::MOST <= OF * TEAM);
    const int teams = (pc.shares + OF - 1) / OF, first = pc.share / OF * OF, n = min(OF, pc.shares - first);
    if (!last_of(&a.count[pc.slot + first], n)) return;
    join_shares<F, D>(a, pc.slot + first, n, 1, pairs, lds, teams == 1, row);
    if (teams == 1 || !last_of(&a.count[Few::SLOTS + Rows::SLOTS + pc.slot], teams)) return;
    join_shares<F, D>(a, pc.slot, teams, OF, pairs, lds, true, row);
}

// The values of a 32-key tile that are no numbers, taken out of it (v: an A operand per granule and 32
// dims) and added to the sums o of those pairs that see the key, `sees` of its index in the tile; through
// `lds`, 64 D B of the wave's own.
template <int D, typename Sees>
__device__ __forceinline__ void add_not_finite(u32x4 (&v)[2][D / 32], f32x16 (&o)[D / 32], uint8_t *lds, int lane, Sees sees) {
    const int l32 = lane & 31, hi = lane >> 5;
    uint16_t *vl = (uint16_t *)lds;  // [key][dim]
    uint32_t keys = 0;
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const int key = 16 * j + 8 * (w >> 1) + 4 * hi + 2 * (w & 1);
#pragma unroll
            for (int dt = 0; dt < D / 32; dt++) {
                const uint32_t x = v[j][dt][w];
                vl[key * D + 32 * dt + l32] = (uint16_t)x;
                vl[(key + 1) * D + 32 * dt + l32] = (uint16_t)(x >> 16);
                const bool a = (x & 0x7f80u) == 0x7f80u, b = (x & 0x7f800000u) == 0x7f800000u;
                keys |= (a ? 1u << key : 0u) | (b ? 2u << key : 0u);
                v[j][dt][w] = x & ((a ? 0u : 0xffffu) | (b ? 0u : 0xffff0000u));
            }
        }
#pragma unroll
    for (int i = 32; i > 0; i >>= 1) keys |= (uint32_t)__shfl_xor((int)keys, i);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll 1
    for (keys = __builtin_amdgcn_readfirstlane(keys); keys; keys &= keys - 1) {
        const int key = __builtin_ctz(keys);
        const bool mine = sees(key);
#pragma unroll
        for (int dt = 0; dt < D / 32; dt++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const u32x2 x = *(const u32x2 *)(vl + key * D + 32 * dt + 8 * e + 4 * hi);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t u = i & 1 ? x[i >> 1] & 0xffff0000u : x[i >> 1] << 16;
                    if (mine && (u & 0x7f800000u) == 0x7f800000u) o[dt][4 * e + i] += __uint_as_float(u);
                }
            }
    }
    __builtin_amdgcn_wave_barrier();
}

constexpr int few_lds(int d) { return 4 * 32 * (d + 4) * 4; }

// A tile of few pairs.
template <int D>
__device__ __forceinline__ void few_pairs(const Attn &a, int item, uint8_t *lds) {
    constexpr int KK = D / 16, DT = D / 32, PITCH = D + 4;
    float *so = (float *)lds;
    __shared__ float sm[4][32], sl[4][32];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int l32 = lane & 31, hi = lane >> 5;

    Piece pc;
    if (!piece_of<Few>(a, item, (int)gridDim.x - a.row_pieces, pc)) return;
    const int r = pc.r, h = pc.h, tile = pc.tile;
    const Req rq = pc.rq;

    // ---- the granules of the wave's next 32 tiles, lane 2 k + j: granule j of tile k (-1: no page) ----
    const int32_t *table = a.tables + (int64_t)r * a.max_pages;
    auto page_at = [&](uint32_t x, uint32_t &k) __attribute__((always_inline)) {
        k = __umulhi(x, a.ps16_magic) + (a.ps16 == 1 ? x : 0);
        return (int64_t)k < a.max_pages ? table[k] : -1;
    };
    // without a window and shares the first ones do not depend on the length: one read less before the keys'
    uint32_t k0 = 0;
    const uint32_t x0 = 2 * (wave + (lane >> 1) * 4) + (lane & 1);
    const bool ahead = !a.window && pc.shares == 1;
    int page0 = -1;
    if (ahead) page0 = page_at(x0, k0);

    // the lane's pair: row i of the request, head h G + hd; its queries' dims 16 kk + 8 hi .. + 7
    const int f = tile * 32 + l32, row = row_of_pair(a, f), hd = f - row * a.G;
    const bool there = row < rq.n;
    bf16x8 qf[KK];
    {
        const uint16_t *src = a.q + (int64_t)(rq.start + (there ? row : 0)) * a.q_row + (int64_t)(h * a.G + (there ? hd : 0)) * a.q_head + 8 * hi;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            u32x4 v = *(const u32x4 *)(src + 16 * kk);
            if (!there) v = u32x4{};
            qf[kk] = __builtin_bit_cast(bf16x8, v);
        }
    }

    const Range g = range_of<KT>(a, rq, tile * 32, 32);
    // the share's tiles: whole rounds
    const int rounds = (g.tiles + 3) / 4;
    const int first = (int)((int64_t)rounds * pc.share / pc.shares) * 4;
    const int last = min((int)((int64_t)rounds * (pc.share + 1) / pc.shares) * 4, g.tiles);
    const int pos = !there ? -1 : max(a.causal ? rq.len - rq.n + row : rq.len - 1, -1);
    const int low = a.window ? pos - a.window : -1;  // sees key j <= pos if j > low or j < g.sk

    int gran = 0;
    auto granule_of = [&](int page, uint32_t x, uint32_t k) __attribute__((always_inline)) {
        return page >= 0 && page < a.pages ? (page * a.Hkv + h) * a.ps16 + (int)(x - k * a.ps16) : -1;
    };
    auto load_granules = [&](int v) __attribute__((always_inline)) {
        const int mine = v + (lane >> 1) * 4;
        gran = -1;
        if (mine < last) {
            const uint32_t x = 2 * tile_at(g, mine) + (lane & 1);
            uint32_t k;
            const int page = page_at(x, k);
            gran = granule_of(page, x, k);
        }
    };
    u32x4 kc[KK], vc[2][DT];
    auto base_of = [&](int gn) __attribute__((always_inline)) { return a.cache + (int64_t)max(gn, 0) * granule_bytes(D); };
    auto load_k = [&](int g0, int g1) __attribute__((always_inline)) {
        const uint8_t *p = (l32 < 16 ? base_of(g0) : base_of(g1)) + hi * 256 + (l32 & 15) * 16;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) kc[kk] = *(const u32x4 *)(p + kk * 512);
    };
    auto load_v = [&](int g0, int g1) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint8_t *p = base_of(j ? g1 : g0) + D * 32 + hi * (D * 16) + l32 * 16;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) vc[j][dt] = *(const u32x4 *)(p + dt * 512);
        }
    };

    f32x16 o[DT] = {};
    float m = -INFINITY, l = 0.f;
    int g0 = -1, g1 = -1, n0 = -1, n1 = -1, k = 0;
    int v = first + wave;
    if (v < last) {
        if (ahead)
            gran = (int)(x0 >> 1) < last ? granule_of(page0, x0, k0) : -1;
        else
            load_granules(v);
        g0 = __builtin_amdgcn_readlane(gran, 0);
        g1 = __builtin_amdgcn_readlane(gran, 1);
        load_k(g0, g1);
        load_v(g0, g1);
    }
    for (; v < last; v += 4) {
        const int key0 = tile_at(g, v) * KT;
        f32x16 s = {};
#pragma unroll
        for (int kk = 0; kk < KK; kk++)
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kc[kk]), qf[kk], s, 0, 0, 0);
        const bool more = v + 4 < last;
        if (more) {
            if (++k == 32) {
                k = 0;
                load_granules(v + 4);
            }
            n0 = __builtin_amdgcn_readlane(gran, 2 * k);
            n1 = __builtin_amdgcn_readlane(gran, 2 * k + 1);
            load_k(n0, n1);
        }

        // every pair that there is sees all of the tile, or some do not (those that are not have queries of 0)
        const bool some = !(key0 + KT - 1 <= g.pos0 && (g0 | g1) >= 0 &&
                            (a.window == 0 || key0 > g.pos1 - a.window || key0 + KT <= g.sk));
        if (some) {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int key = key0 + 8 * (e >> 2) + 4 * hi + (e & 3);
                const bool ok = key <= pos && (key > low || key < g.sk) && (e < 8 ? g0 : g1) >= 0;
                s[e] = ok ? s[e] : -INFINITY;
            }
        }
        float mx = s[0];
#pragma unroll
        for (int e = 1; e < 16; e++) mx = fmaxf(mx, s[e]);
        mx = fmaxf(fmaxf(mx, __shfl_xor(mx, 32)), m);
        if (__ballot(mx > m)) {
            // a pair without a visible key so far has sums of 0
            const float al = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mx) * a.sl2);
            m = mx;
            l *= al;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[dt][e] *= al;
        }
        const float c = mx == -INFINITY ? 0.f : -mx * a.sl2;
        float sum = 0.f;
        uint32_t p[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * e], a.sl2, c));
            const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * e + 1], a.sl2, c));
            sum += x;
            sum += y;
            p[e] = pack_bf16x2(x, y);
        }
        l += sum;

        bf16x8 pf[2];
#pragma unroll
        for (int j = 0; j < 2; j++) pf[j] = __builtin_bit_cast(bf16x8, u32x4{p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]});
        // where not every pair sees all of it, values that are no numbers (0 times them is NaN) go to
        // those that see them by themselves
        if (some) {
            uint32_t mag = 0;
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int w = 0; w < 4; w++) mag = magnitude2(mag, vc[j][dt][w]);
            if (__builtin_expect(__ballot(not_finite2(mag)) != 0, 0))
                add_not_finite<D>(vc, o, (uint8_t *)(so + wave * 32 * PITCH), lane, [&](int i) {
                    const int key = key0 + i;
                    return key <= pos && (key > low || key < g.sk) && (i < 16 ? g0 : g1) >= 0;
                });
        }
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
                o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, vc[j][dt]), pf[j], o[dt], 0, 0, 0);
        if (more) load_v(n0, n1);
        g0 = n0;
        g1 = n1;
    }

    // ---- the four waves' sums ----
    m = lowest_of<KT, 4>(a, table, g, first + wave, last, m, pos, low, g.sk);
    l += __shfl_xor(l, 32);
    if (hi == 0) {
        sm[wave][l32] = m;
        sl[wave][l32] = l;
    }
    float *mine = so + (wave * 32 + l32) * PITCH + 4 * hi;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            *(f32x4 *)(mine + 32 * dt + 8 * e) = f32x4{o[dt][4 * e], o[dt][4 * e + 1], o[dt][4 * e + 2], o[dt][4 * e + 3]};
    __syncthreads();
    const int pairs = min(rq.n * a.G - tile * 32, 32), pr = tid / 8;  // eight threads a pair
    auto row_of = [&](int p) __attribute__((always_inline)) {
        const int at = row_of_pair(a, tile * 32 + p), hd = tile * 32 + p - at * a.G;
        return a.out + ((int64_t)(rq.start + at) * a.Hkv * a.G + h * a.G + hd) * D;
    };
    const Part pb(slot_at<Few, D>(a, pc.slot + pc.share), slot_floats<Few, D>());
    if (pr < pairs) {
        const float mm = fmaxf(fmaxf(sm[0][pr], sm[1][pr]), fmaxf(sm[2][pr], sm[3][pr]));
        float ll = 0.f, fac[4];
#pragma unroll
        for (int w = 0; w < 4; w++) {
            fac[w] = sm[w][pr] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((sm[w][pr] - mm) * a.sl2);
            ll += sl[w][pr] * fac[w];
        }
        const float inv = mm == -INFINITY ? 0.f : 1.0f / ll;  // a pair that sees no key gives zeros
        if (pc.shares > 1 && (tid & 7) == 0) pb.put2(32 * D + 2 * pr, mm, ll);
        uint16_t *dst = row_of(pr);
#pragma unroll
        for (int e = 0; e < D / 32; e++) {
            const int d = (tid & 7) * 4 + 32 * e;
            f32x4 x{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const f32x4 y = *(const f32x4 *)(so + (w * 32 + pr) * PITCH + d);
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] += y[i] * fac[w];
            }
            if (pc.shares > 1)
                pb.put4(pr * D + d, x);
            else
                *(u32x2 *)(dst + d) = u32x2{pack_bf16x2(x[0] * inv, x[1] * inv), pack_bf16x2(x[2] * inv, x[3] * inv)};
        }
    }
    if (pc.shares > 1) arrive<Few, D>(a, pc, pairs, so, row_of);
}

// ---- many pairs ----

// 4 KB of consecutive memory, 64 lanes of 16 B four times, into LDS (from `dst`, uniform, on) without
// registers. The caller waits (lds_wait). In assembly, where the compiler does not see that LDS is
// written: it would have every later read of LDS wait for these loads, those of the other stage too.
__device__ __forceinline__ void load_lds_4k(const uint8_t *src, uint8_t *dst) {
    const uint32_t at = (uint32_t)(uintptr_t)(lds_ptr_t)dst;
    uint32_t m0;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %1\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %2, off\n\t"
        "global_load_lds_dwordx4 %2, off offset:%3\n\t"
        "global_load_lds_dwordx4 %2, off offset:%4\n\t"
        "global_load_lds_dwordx4 %2, off offset:%5\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(m0)
        : "s"(__builtin_amdgcn_readfirstlane(at)), "v"(src), "i"(1 << 10), "i"(2 << 10), "i"(3 << 10)
        : "memory");
}
__device__ __forceinline__ void lds_wait() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

constexpr int rows_lds(int d) { return 8 * (int)granule_bytes(d); }

// A tile of 128 pairs, a wave 32 of them: 64-key tiles go straight from the pages into LDS, a granule a
// wave, the next one while this one is multiplied. K operands are read there conflict-free (paged.h).
// The reference point of a pair's exponentials follows its maximum where that grew by more than 2^8.
template <int D>
__device__ __forceinline__ void many_pairs(const Attn &a, int item, uint8_t *lds) {
    constexpr int KK = D / 16, DT = D / 32, KEYS = 64;
    constexpr int GB = (int)granule_bytes(D), STAGE = 4 * GB;
    constexpr float LAG = 8.f;
    constexpr int ODD = 1 << 30;
    __shared__ int info[2][4];  // a stage's granules: -1 without a page, ODD where values were taken out
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int l32 = lane & 31, hi = lane >> 5;

    Piece pc;
    if (!piece_of<Rows>(a, item, a.row_pieces, pc)) return;
    const int r = pc.r, h = pc.h, f0 = pc.tile * Rows::TM;
    const Req rq = pc.rq;
    const Range g = range_of<KEYS>(a, rq, f0, Rows::TM);
    const int first = (int)((int64_t)g.tiles * pc.share / pc.shares);
    const int last = (int)((int64_t)g.tiles * (pc.share + 1) / pc.shares);

    // the wave's pairs
    const int pairs = min(rq.n * a.G - f0, Rows::TM);
    const Range w = range_of<KEYS>(a, rq, f0 + 32 * wave, 32);
    const bool any = 32 * wave < pairs;
    const int f = f0 + 32 * wave + l32, row = row_of_pair(a, f), hd = f - row * a.G;
    const bool there = row < rq.n;
    const int pos = !there ? -1 : max(a.causal ? rq.len - rq.n + row : rq.len - 1, -1);
    const int low = a.window ? pos - a.window : -1;      // sees key j <= pos if j > low or j < sk
    const int low0 = a.window ? w.pos0 - a.window : -1, sk = a.window ? a.sinks : 0;

    // ---- tiles from the pages: the wave's granule of the next 64 tiles, a lane each ----
    const int32_t *table = a.tables + (int64_t)r * a.max_pages;
    int gran = -1, k = 0, here = -1;
    auto load_granules = [&](int v) __attribute__((always_inline)) {
        gran = -1;
        if (v + lane < last) {
            const uint32_t x = 4 * tile_at(g, v + lane) + wave;
            const uint32_t k = __umulhi(x, a.ps16_magic) + (a.ps16 == 1 ? x : 0);
            if ((int64_t)k < a.max_pages) {
                const int page = table[k];
                if (page >= 0 && page < a.pages) gran = (page * a.Hkv + h) * a.ps16 + (int)(x - k * a.ps16);
            }
        }
    };
    auto load_tile = [&](int v, auto stage) __attribute__((always_inline)) {
        constexpr int ST = decltype(stage)::value;
        if (k == 64) {
            k = 0;
            load_granules(v);
        }
        here = __builtin_amdgcn_readlane(gran, k++);
        const uint8_t *src = a.cache + (int64_t)max(here, 0) * GB + lane * 16;
#pragma unroll
        for (int i = 0; i < GB / 4096; i++) load_lds_4k(src + i * 4096, lds + ST * STAGE + wave * GB + i * 4096);
        info[ST][wave] = here;
    };
    // The wave's granule of tile v is there. Where not every pair of the workgroup sees all of the tile, values
    // that are no numbers are taken out (0 times them is NaN); those that some pairs see go to these by
    // themselves below.
    auto clean = [&](int key0, auto stage) __attribute__((always_inline)) {
        constexpr int ST = decltype(stage)::value;
        if (here >= 0 && key0 + KEYS - 1 <= g.pos0 && (a.window == 0 || key0 > g.pos1 - a.window || key0 + KEYS <= sk)) return;
        u32x4 *const mine = (u32x4 *)(lds + ST * STAGE + wave * GB + D * 32 + lane * 16);
        uint32_t mag = 0;
#pragma unroll
        for (int i = 0; i < D / 32; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) mag = magnitude2(mag, mine[64 * i][j]);
        if (__builtin_expect(__ballot(not_finite2(mag)) == 0, 1)) return;
        const int above = a.window ? g.pos0 - a.window : -1;
        bool odd = false;
#pragma unroll 1
        for (int i = 0; i < D / 32; i++) {
            // 64 lanes: a half's keys of 64 dims
            const int half = i / (D / 64);
            u32x4 x = mine[64 * i];
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int key = key0 + 16 * wave + 8 * (j >> 1) + 4 * half + 2 * (j & 1) + e;
                    const uint32_t big = e ? 0x7f800000u : 0x7f80u;
                    if ((x[j] & big) != big) continue;
                    odd = odd || (here >= 0 && key <= g.pos1 && (key > above || key < sk));
                    x[j] &= e ? 0xffffu : 0xffff0000u;
                }
            mine[64 * i] = x;
        }
        if (__ballot(odd)) info[ST][wave] = here | ODD;
    };
    if (first < last) {
        load_granules(first);
        load_tile(first, std::integral_constant<int, 0>{});
    }

    bf16x8 qf[KK];
    {
        const uint16_t *src = a.q + (int64_t)(rq.start + (there ? row : 0)) * a.q_row + (int64_t)(h * a.G + (there ? hd : 0)) * a.q_head + 8 * hi;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            u32x4 x = *(const u32x4 *)(src + 16 * kk);
            if (!there) x = u32x4{};
            qf[kk] = __builtin_bit_cast(bf16x8, x);
        }
    }

    f32x16 o[DT] = {};
    float m = -INFINITY, mc = 0.f, l[4] = {};
    const uint8_t *kl = lds + (l32 >> 4) * GB + hi * 256 + (l32 & 15) * 16;  // + half, dims
    const uint8_t *vl = lds + D * 32 + hi * (D * 16) + l32 * 16;             // + granule, dims

    auto step = [&](int v, auto stage) __attribute__((always_inline)) {
        constexpr int ST = decltype(stage)::value;
        const int key0 = tile_at(g, v) * KEYS;
        lds_wait();
        clean(key0, stage);
        __syncthreads();
        if (v + 1 < last) load_tile(v + 1, std::integral_constant<int, ST ^ 1>{});
        // no pair of the wave sees any of it
        if (!any || key0 > w.pos1 || (a.window && key0 + KEYS - 1 <= low0 && key0 >= sk)) return;
        const int about = info[ST][lane & 3];

        f32x16 s[2] = {};
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int kk = 0; kk < KK; kk++)
                s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8 *)(kl + ST * STAGE + b * 2 * GB + kk * 512), qf[kk], s[b], 0, 0, 0);
        // every pair sees all of it, or some do not
        const uint32_t gone = (uint32_t)__ballot(about < 0) & 15u;
        if (key0 + KEYS - 1 > w.pos0 || gone || (a.window && key0 <= w.pos1 - a.window && key0 + KEYS > sk)) {
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int key = key0 + 32 * b + 8 * (e >> 2) + 4 * hi + (e & 3);
                    const int ok = (int)(key <= pos) & ((int)(key > low) | (int)(key < sk)) & (int)(~gone >> (2 * b + (e >> 3)));
                    s[b][e] = ok & 1 ? s[b][e] : -INFINITY;
                }
        }
        float m0 = s[0][0], m1 = s[1][0];
#pragma unroll
        for (int e = 1; e < 16; e++) {
            m0 = fmaxf(m0, s[0][e]);
            m1 = fmaxf(m1, s[1][e]);
        }
        float mx = fmaxf(m0, m1);
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        if (__ballot((mx - m) * a.sl2 > LAG)) {  // (a pair without a visible key yet: NaN or infinity)
            const float top = fmaxf(mx, m);
            const float al = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - top) * a.sl2);
            m = top;
            mc = m == -INFINITY ? 0.f : -m * a.sl2;
#pragma unroll
            for (int i = 0; i < 4; i++) l[i] *= al;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[dt][e] *= al;
        }
#pragma unroll
        for (int b = 0; b < 2; b++) {
            uint32_t p[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][2 * e], a.sl2, mc));
                const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][2 * e + 1], a.sl2, mc));
                l[2 * b] += x;
                l[2 * b + 1] += y;
                p[e] = pack_bf16x2(x, y);
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const bf16x8 pf = __builtin_bit_cast(bf16x8, u32x4{p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]});
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8 *)(vl + ST * STAGE + (2 * b + j) * GB + dt * 512), pf, o[dt], 0, 0, 0);
            }
        }
        if (__builtin_expect(__ballot(about >= ODD) != 0, 0)) {
#pragma unroll 1
            for (int i = 0; i < KEYS; i++) {
                const int key = key0 + i, from = __builtin_amdgcn_readlane(about, i >> 4);
                if (from < ODD) continue;
                const bool sees = key <= pos && (key > low || key < sk);
                const uint8_t *src = a.cache + (int64_t)(from - ODD) * GB + granule_v(D, i & 15, 0);
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const uint32_t u = (uint32_t)*(const uint16_t *)(src + (32 * dt + 8 * (e >> 2) + 4 * hi + (e & 3)) * 16) << 16;
                        if (sees && (u & 0x7f800000u) == 0x7f800000u) o[dt][e] += __uint_as_float(u);
                    }
            }
        }
    };
    for (int v = first; v < last; v += 2) {
        step(v, std::integral_constant<int, 0>{});
        if (v + 1 < last) step(v + 1, std::integral_constant<int, 1>{});
    }

    m = lowest_of<KEYS, 1>(a, table, g, first, last, m, pos, low, sk);
    float lsum = l[0] + l[1] + l[2] + l[3];
    lsum += __shfl_xor(lsum, 32);
    auto row_of = [&](int p) __attribute__((always_inline)) {
        const int at = row_of_pair(a, f0 + p), head = f0 + p - at * a.G;
        return a.out + ((int64_t)(rq.start + at) * a.Hkv * a.G + h * a.G + head) * D;
    };
    const int p = 32 * wave + l32;
    if (pc.shares == 1) {
        // through LDS, the wave's 32 rows of D in a pitch of D + 8, so that a store covers whole rows
        __syncthreads();
        constexpr int PITCH = 2 * D + 16;
        uint8_t *mine = lds + wave * 32 * PITCH;
        const float inv = m == -INFINITY ? 0.f : 1.0f / lsum;  // a pair that sees no key gives zeros
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                *(u32x2 *)(mine + l32 * PITCH + (32 * dt + 8 * e + 4 * hi) * 2) =
                    u32x2{pack_bf16x2(o[dt][4 * e] * inv, o[dt][4 * e + 1] * inv), pack_bf16x2(o[dt][4 * e + 2] * inv, o[dt][4 * e + 3] * inv)};
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        constexpr int LPR = D / 8;  // lanes a row
#pragma unroll
        for (int i = 0; i < 32 * LPR / 64; i++) {
            const int q = i * (64 / LPR) + lane / LPR;
            if (32 * wave + q < pairs)
                *(u32x4 *)(row_of(32 * wave + q) + lane % LPR * 8) = *(const u32x4 *)(mine + q * PITCH + lane % LPR * 16);
        }
        return;
    }
    if (there) {
        const Part pb(slot_at<Rows, D>(a, pc.slot + pc.share), slot_floats<Rows, D>());
        if (hi == 0) pb.put2(Rows::TM * D + 2 * p, m, lsum);
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                pb.put4(wave * (32 * D) + (4 * dt + e) * 256 + lane * 4, f32x4{o[dt][4 * e], o[dt][4 * e + 1], o[dt][4 * e + 2], o[dt][4 * e + 3]});
    }
    arrive<Rows, D>(a, pc, pairs, (float *)lds, row_of);
}

template <int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void paged_tokens_kernel(const Attn a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[few_lds(D)];
    few_pairs<D>(a, blockIdx.x, lds);
}
// Pieces of requests with many pairs and with few in turn, as many of each as there are CUs, as long as there are
// both: the first are bound by the matrix pipe, the others by memory, and a CU has one of each (two chunks
// of 517 rows and 30 single tokens, 59 and 81 us by themselves: 143 one after the other, 135 in turn).
template <int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void paged_rows_kernel(const Attn a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[few_lds(D) > rows_lds(D) ? few_lds(D) : rows_lds(D)];
    const int turn = a.turn, at = blockIdx.x / turn, rows = a.row_pieces / turn, both = min(rows, (int)(gridDim.x / turn) - rows);
    const bool many = at < 2 * both ? !(at & 1) : rows > both;
    const int item = (at < 2 * both ? at >> 1 : at - both) * turn + blockIdx.x % turn;
    if (many)
        many_pairs<D>(a, item, lds);
    else
        few_pairs<D>(a, item, lds);
}

}  // namespace

size_t paged_attention_scratch(int d) {
    return PAGED_COUNTER_BYTES + ((size_t)Few::SLOTS * Few::TM + (size_t)Rows::SLOTS * Rows::TM) * (d + 2) * 4;
}

hipError_t launch_paged_attention(const PageDims &d, const uint8_t *layer, const PagedAttnArgs &x, void *scratch,
                                  hipStream_t stream) {
    if (x.rows <= 0 || x.requests <= 0) return hipSuccess;
    const int64_t g = x.heads / d.kv_heads, cap = std::min<int64_t>(std::min<int64_t>(x.max_pages, 0x7fffffff) * d.page_size, 0x7fffffff - 64);
    const int ps16 = d.page_size / 16;
    Attn a{x.q, x.q_row, x.q_head, layer, d.pages, x.tables, x.max_pages, x.lengths, x.starts, (int32_t)x.requests,
           (int32_t)x.rows, d.kv_heads, (int32_t)g, ps16, (uint32_t)(((1ull << 32) + ps16 - 1) / ps16),
           (int32_t)cap, x.causal, (int32_t)std::min<int64_t>(x.window, 0x7fffffff),
           (int32_t)std::min<int64_t>(x.sinks, 0x7fffffff), x.scale * 1.4426950408889634f, x.out, nullptr, nullptr, 0, 0,
           g > 1 ? ~0ull / (uint64_t)g + 1 : 0, {}};
    const int cus = std::max(device_cu_count(), 1);
    a.want[0] = std::min(Few::ON_CU * cus, Few::SLOTS);
    a.want[1] = std::min(Rows::ON_CU * cus, Rows::SLOTS);
    // Workgroups: of a request with few pairs one for each key head, of one with many at most a tile more
    // than its pairs fill, and the shares. Without starts every request has g pairs.
    const bool rows = x.starts ? x.rows * g > FEW_PAIRS : g > FEW_PAIRS, few = g <= FEW_PAIRS;
    int64_t many = rows ? (x.rows * g / Rows::TM + std::min(x.requests, x.rows)) * d.kv_heads : 0;
    int64_t tokens = few ? std::min(x.requests, x.rows) * d.kv_heads : 0;
    if (cap > std::min(Few::GRAIN * Few::ROUND, Rows::GRAIN * Rows::ROUND)) {
        a.count = (uint32_t *)scratch;
        a.part = (float *)((char *)scratch + PAGED_COUNTER_BYTES);
        const int64_t keys = x.window ? std::min<int64_t>(cap, std::min<int64_t>(x.sinks, cap) + std::min<int64_t>(x.window, cap) + 512) : cap;
        many = std::min(many * (1 + keys / (Rows::GRAIN / 2 * Rows::ROUND)), many + 2 * a.want[1]);
        tokens = std::min(tokens * (1 + keys / (Few::GRAIN / 2 * Few::ROUND)), tokens + a.want[0]);
    }
    a.turn = (cus + 7) / 8 * 8;
    many = (many + a.turn - 1) / a.turn * a.turn;
    if (many) tokens = (tokens + a.turn - 1) / a.turn * a.turn;
    if (many + tokens >= (int64_t)1 << 24) return hipErrorInvalidValue;
    a.row_pieces = (int32_t)many;
    const unsigned grid = (unsigned)(many + tokens);
    if (d.head_dim == 128) {
        if (many)
            paged_rows_kernel<128><<<grid, 256, 0, stream>>>(a);
        else
            paged_tokens_kernel<128><<<grid, 256, 0, stream>>>(a);
    } else if (d.head_dim == 64) {
        if (many)
            paged_rows_kernel<64><<<grid, 256, 0, stream>>>(a);
        else
            paged_tokens_kernel<64><<<grid, 256, 0, stream>>>(a);
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace qimm
