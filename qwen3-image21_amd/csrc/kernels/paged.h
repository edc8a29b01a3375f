// Layout of the paged K/V cache (bf16) and the arguments of its kernels.
//
// A layer is [page][kv head][page_size / 16] granules of 16 keys of one head, 64 D bytes each:
//   K  [D / 8][16 keys][8 dims]
//   V  [2][D][8 keys], half g holding keys 4 g .. 4 g + 3 and 8 + 4 g .. 8 + 4 g + 3
// so that the operands of v_mfma_f32_32x32x16_bf16 are 16 B a lane and 512 B or more of consecutive
// lanes, from memory and from an LDS copy (where 16 lanes then cover all 64 banks once): K rows
// m = 0 .. 31 are 32 keys in order, which leaves lane (q, g) of S^T = K Q^T with keys
// 8 i + 4 g + e in registers 4 i + e, and registers 8 j .. 8 j + 7 are the B operand of
// O^T = V^T P^T for granule j in the order that V has its keys.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.h"

namespace qimm {

__host__ __device__ constexpr int64_t granule_bytes(int d) { return 64 * (int64_t)d; }
// byte of (key k, dim) of a granule's halves
__device__ __forceinline__ int granule_k(int k, int dim) { return (dim >> 3) * 256 + k * 16 + (dim & 7) * 2; }
__device__ __forceinline__ int granule_v(int d, int k, int dim) {
    return d * 32 + ((k >> 2) & 1) * d * 16 + dim * 16 + ((k >> 3) * 4 + (k & 3)) * 2;
}

}  // namespace qimm
