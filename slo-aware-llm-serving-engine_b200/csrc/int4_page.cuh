// Layout of the 4-bit KV pool.
//
// One side (K or V) of a pool is uint8 [num_blocks, num_kv_heads, block_size * 72]:
// head-major inside a block, so that one head's tokens are contiguous.  A (block,
// head) run is block_size / 64 tiles of 4608 bytes; a tile holds 64 tokens as
//   64 x 64 B   codes: 128 unsigned 4-bit codes of a token, dim 2i in the low and
//               2i + 1 in the high half of byte i of its group's 32 bytes; the
//               row's sixteen 32-bit words alternate between the two groups (stored
//               word 2i + g is word i of group g), which gives a decode lane one
//               16-byte (K) or 8-byte (V) load with dims of both groups
//   64 x 8 B    (scale, minimum) of group 0 (dims 0-63) and of group 1 (64-127), bf16
// value = minimum + scale * code.  bf16 parameters keep the whole fp32 range; a
// bf16 group's minimum is stored exactly.  A tile is one bulk copy.
#pragma once

#include "common.cuh"

namespace slokv {
namespace kv4 {

constexpr int kHeadDim = 128;
constexpr int kTileTokens = 64;
constexpr int kCodeRow = 64;                              // code bytes of a token
constexpr int kParamRow = 8;                              // scale / minimum bytes of a token
constexpr int kRowBytes = kCodeRow + kParamRow;           // 72
constexpr int kParamOff = kTileTokens * kCodeRow;         // 4096: parameters of a tile
constexpr int kTileBytes = kTileTokens * kRowBytes;       // 4608

// Byte offset of token `off`'s codes inside its (block, head) run, and of its
// parameters.
__device__ __forceinline__ int64_t code_offset(int32_t off) {
  return static_cast<int64_t>(off / kTileTokens) * kTileBytes + (off % kTileTokens) * kCodeRow;
}
__device__ __forceinline__ int64_t param_offset(int32_t off) {
  return static_cast<int64_t>(off / kTileTokens) * kTileBytes + kParamOff +
         (off % kTileTokens) * kParamRow;
}

// The two bf16 of a parameter word: scale in the low half, minimum in the high.
__device__ __forceinline__ float scale_of(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float min_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

}  // namespace kv4
}  // namespace slokv
