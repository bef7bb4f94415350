// 8-bit floating-point rows: codes in e4m3 (a sign, 4 bits of exponent, 3 of mantissa, largest 448), and for each block of
// 128 elements along a row a byte with the power of two that they count in: element = code * 2^(byte - 127), the smallest for
// which the block's largest magnitude is at most 448 units (not below 2^-127). 255 marks a block that held an infinity or
// NaN: all of it is NaN.
//
// The bytes lie as the tensor core takes them: 128 rows and 4 blocks in 512 bytes, row r of the 128 at 16 (r % 32) +
// 4 (r / 32), its four blocks one after the other.
#pragma once
#include "rows.cuh"

namespace flb {
namespace fp8 {

constexpr int kBlock = 128;      // elements of a row that share a power of two; rows, and blocks times 32, of a tile of bytes
constexpr int kTileBytes = 512;

__host__ __device__ inline int64_t blocks_of(int64_t K) { return (K + kBlock - 1) / kBlock; }
__host__ __device__ inline int64_t quads_of(int64_t K) { return (blocks_of(K) + 3) / 4; }
__host__ __device__ inline int64_t exps_bytes(int64_t R, int64_t K) { return blocks_of(R) * quads_of(K) * kTileBytes; }
__host__ __device__ inline int64_t exp_at(int64_t row, int64_t block, int64_t quads) {
  return (row / kBlock * quads + block / 4) * kTileBytes + row % 32 * 16 + row / 32 % 4 * 4 + block % 4;
}

// The byte of a block whose largest magnitude has these float32 bits: 448 = 1.75 * 2^8
__device__ __forceinline__ int unit_of(uint32_t top) {
  if (top >= 0x7f800000u) return 255;
  return max(0, (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0));
}
// what brings an element into units: 2^(127 - byte), exact
__device__ __forceinline__ float inverse_of(int unit) { return __uint_as_float((uint32_t)(254 - min(unit, 253)) << 23); }

// two codes, of a in the low byte
__device__ __forceinline__ uint32_t code2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d) { return code2(a, b) | code2(c, d) << 16; }

}  // namespace fp8
}  // namespace flb
