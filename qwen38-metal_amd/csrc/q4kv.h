// Layout of the 4-bit KV cache, shared by the kernels that write and read it.
//
// A token's keys (and values) of one KV head are groups of 64 elements, each
// with a bf16 scale s and offset m: x ~ s c + m, c a whole number in -8..7.
// The blocks of a (page, KV head), 18 Dp bytes in one piece, are what a wave of
// the decode kernel takes with one coalesced load each, lane by lane, straight
// into matrix operands.  With lane = 16 kq + (token or d) % 16, kq = 0..3:
//   K, 8 Dp bytes: the lane of (token, kq) holds d = 64 g + 16 kq .. + 15 of every
//     group g, two words each; word w is d = 64 g + 16 kq + 8 w .. + 7, element e
//     of it in nibble (e >> 1) + 4 (e & 1), as c + 8: masks of one shifted word are
//     pairs (e, e + 1) of bf16 operands.
//   V, 8 Dp bytes: the lane of (d % 16, kq) holds tokens 4 kq .. 4 kq + 3 of its d's;
//     word j holds d / 16 = 2 j and 2 j + 1, token r of the four in nibble
//     2 (d / 16 % 2) + (r >> 1) + 4 (r & 1), as c + 8: pairs of tokens again.
//   Words 0..3 of a lane are 16 bytes, words 4..7 (Dp = 256) the 16 bytes 1024
//   further; with Dp = 64 a lane has two words.
//   Scales, 2 Dp bytes: token by token a word per group of K, then of V, s in its low
//     half and m in its high one.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qm {

constexpr uint32_t kQ4KvGroup = 64;

__host__ __device__ constexpr uint32_t q4kv_block_bytes(uint32_t dp) { return 18 * dp; }
__host__ __device__ constexpr uint32_t q4kv_v_bytes(uint32_t dp) { return 8 * dp; }       // where V starts
__host__ __device__ constexpr uint32_t q4kv_scale_bytes(uint32_t dp) { return 16 * dp; }  // where the scales start

// Byte of word w (0 .. dp / 32 - 1) of a lane within the K or V part.
__host__ __device__ constexpr uint32_t q4kv_lane_word(uint32_t dp, uint32_t lane, uint32_t w) {
  return dp == 64 ? 8 * lane + 4 * w : 1024 * (w / 4) + 16 * lane + 4 * (w % 4);
}
// Nibble of (token, d): byte of its word within the K part, and bit.
__host__ __device__ constexpr uint32_t q4kv_k_word(uint32_t dp, uint32_t token, uint32_t d) {
  return q4kv_lane_word(dp, 16 * (d % 64 / 16) + token, 2 * (d / 64) + d % 16 / 8);
}
__host__ __device__ constexpr uint32_t q4kv_k_bit(uint32_t d) { return 4 * ((d % 8 >> 1) + 4 * (d & 1)); }
// The same of V.
__host__ __device__ constexpr uint32_t q4kv_v_word(uint32_t dp, uint32_t token, uint32_t d) {
  return q4kv_lane_word(dp, 16 * (token / 4) + d % 16, d / 32);
}
__host__ __device__ constexpr uint32_t q4kv_v_bit(uint32_t token, uint32_t d) {
  return 4 * (2 * (d / 16 % 2) + (token % 4 >> 1) + 4 * (token & 1));
}
// Index of the scale word of (kind: 0 K, 1 V; group; token).
__host__ __device__ constexpr uint32_t q4kv_scale_word(uint32_t dp, uint32_t kind, uint32_t group, uint32_t token) {
  return dp / 32 * token + dp / 64 * kind + group;
}

}  // namespace qm
