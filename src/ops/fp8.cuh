// The 8-bit format of this framework: e4m3 values with one power of two for each block of 128.
//
// A matrix [rows, cols] is rows of cols values, filled with zeros to a multiple of 128, and scales: the byte of row r and block k (128 columns) lies at
// [r / 128][k / 4][r % 32][r / 32 % 4][k % 4].  512 bytes of it, 128 rows by 4 blocks, are what one tcgen05.cp brings into TMEM, where the MMA multiplies by
// 2^(byte - 127) itself: no product is scaled by a thread, and a power of two loses nothing (a scale that is not one would round every value twice).
// A byte is the smallest for which the block's largest finite magnitude is at most 448 = 1.75 * 2^8; blocks of zeros, and what is beyond the matrix, have 1.
#pragma once
#include <cuda_fp8.h>
#include "ops_common.cuh"

namespace piccl_ops {

// bits of |x|, 0 for what is not finite
__device__ __forceinline__ uint32_t finite_bits(float x) { const uint32_t u = __float_as_uint(x) & 0x7fffffffu; return u < 0x7f800000u ? u : 0u; }
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  const int e = (int)((amax_bits + 0x1fffffu) >> 23) - 8;      // carries into the exponent above a mantissa of 1.75
  return e < 1 ? 1u : (uint32_t)e;
}
__device__ __forceinline__ float scale_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }      // 2^(127 - byte), always a normal number
__device__ __forceinline__ float scale_value(uint32_t byte) { return __uint_as_float(byte << 23); }                   // 2^(byte - 127)
__device__ __forceinline__ size_t scale_at(long long row, int block, int blocks4) {
  return (((size_t)(row >> 7) * blocks4 + (block >> 2)) * 32 + (row & 31)) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}
// Two values that are at most 448 in magnitude, or not finite: those become NaN (cvt would take infinities for 448).
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

}  // namespace piccl_ops
