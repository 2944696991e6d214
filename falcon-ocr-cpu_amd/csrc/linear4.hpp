// The device layout of a matrix of 4-bit codes (Linear with bits 4), shared by
// its decode GEMV (gemv_i4.hip) and the kernels that read it back.
//
// Codes c in -8..7 stand in tiles of 16 output channels x 128 columns of 1 KB:
// lane l of a wave holds channel l % 16 and, of each 64-column half, the 16
// columns 16 (l / 16) .. + 15, 8 bytes of its 16-byte chunk per half. Byte b
// of word w of a half holds column 8 w + b in its low nibble and 8 w + 4 + b in
// its high one, so (word << 4) & 0xf0f0f0f0 and word & 0xf0f0f0f0 are the codes
// of four consecutive columns as signed bytes, times 16: the operand of the
// 16 x 16 x 64 INT8 matrix instruction in two or three operations per eight
// codes. Scales: [tile][128-column step][its groups][16 channels]. Channels past
// out and columns past in hold zeros.
#pragma once

#include "focr_internal.hpp"

namespace focr {
namespace linear4 {

constexpr int kTile = 16;   // output channels of a tile
constexpr int kStep = 128;  // columns of a tile's 1 KB

__host__ __device__ inline size_t steps_of(size_t k) { return (k + kStep - 1) / kStep; }
__host__ __device__ inline size_t tiles_of(size_t n) { return (n + kTile - 1) / kTile; }

// The code of one weight.
__device__ __forceinline__ int code_at(const uint8_t *tiles, size_t steps, size_t row, size_t col) {
  const size_t step = col / kStep;
  const int in = static_cast<int>(col % kStep), half = in / 64, j = in % 16, lane = (in % 64) / 16 * 16 + static_cast<int>(row % kTile);
  const uint8_t byte = tiles[((row / kTile * steps + step) * 64 + lane) * 16 + half * 8 + j / 8 * 4 + j % 4];
  const int nibble = j % 8 >= 4 ? byte >> 4 : byte & 15;
  return (nibble ^ 8) - 8;
}

__device__ __forceinline__ float scale_at(const float *scales, size_t steps, size_t group, size_t row, size_t col) {
  const size_t per = kStep / group;  // groups of a step
  return scales[((row / kTile * steps + col / kStep) * per + col % kStep / group) * kTile + row % kTile];
}

}  // namespace linear4
}  // namespace focr
