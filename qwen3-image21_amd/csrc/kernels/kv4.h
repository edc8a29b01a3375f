// Device layout of the prefix cache held in 4 bits (kv4.hip writes and reads it
// back, attn4.hip multiplies it as it lies).
#pragma once

#include "device_common.h"

namespace qimm {

// Blocks of 32 values with one power of two 2^s: e2m1 codes (0, 0.5, 1, 1.5, 2,
// 3, 4, 6 and their negatives), s as a byte s + 127. A key's block runs along 32
// of its dimensions; a value's along 32 consecutive keys of one dimension. Both
// are the contraction of their product, so v_mfma_scale_f32_16x16x128_f8f6f4
// takes codes and scale bytes from memory with no decoding in between.
//
// One (batch, head) is tiles of 128 keys, each 17408 contiguous bytes in the
// order in which a wave's lanes read the operands, lane = 16 lg + l16:
//   K codes  [i < 8][lane][16 B]: key kv4_key(i, l16), dimensions 32 lg + 0..31
//            (low nibble first)
//   V codes  [j < 8][lane][16 B]: dimension 16 j + l16, keys 32 lg + 0..31
//   K scales [i / 4][lane][4 B]: byte i % 4; V scales [j / 4][lane][4 B]
// An e4m3 operand of that product holds, in lane (l16, lg), contraction indices
// 16 lg + 0..15 and 64 + 16 lg + 0..15 (an e2m1 operand 32 lg + 0..31; both checked
// on the device). With this order of the keys the lane's scores of K Q^T, register
// r of product i < 4 for key 16 lg + 4 i + r and of product 4 + i for key 64 + 16 lg
// + 4 i + r, are the keys of its operand in V^T P^T: probabilities stay in their lane.
constexpr int KV4_KEYS = 128;
constexpr int KV4_V = 8192, KV4_KS = 16384, KV4_VS = 16896;
constexpr int KV4_TILE = 17408;

__device__ __forceinline__ int kv4_key(int i, int l16) { return 64 * (i >> 2) + 16 * (l16 >> 2) + 4 * (i & 3) + (l16 & 3); }

}  // namespace qimm
