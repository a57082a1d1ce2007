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

// fp8_few.cu: products of at most 32 rows
bool fp8_few_takes(int M, int N, long long K, bool rounded);
int fp8_few(const bf16* x, long long stride, const void* a, const void* sa, const void* b, const void* sb, const void* bias, void* out, int f32, int M, int N, int K, void* stream);

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
// Four values that are at most 448 in magnitude, or NaN (infinities would be taken for 448: no_inf)
__device__ __forceinline__ uint32_t e4m3_four(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}" : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

// Eight values of a row as they lie in memory, and their magnitudes' bits: bf16 in pairs, 16 bits each, fp32 one by one.  A maximum over these counts values that are not finite; where it says
// that there are some (a bit pattern from `kInf` on), the maximum is taken again without them.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
template <typename T> struct Eight;
template <> struct Eight<bf16> {
  static constexpr int W = 4;                       // words
  uint32_t w[4];
  __device__ __forceinline__ void load(const bf16* p) { const uint4 u = *reinterpret_cast<const uint4*>(p); w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w; }
  __device__ __forceinline__ void set(int e, const bf16* p) { w[e >> 1] |= (uint32_t)*reinterpret_cast<const uint16_t*>(p) << (16 * (e & 1)); }
  __device__ __forceinline__ float at(int e) const { return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16); }
  static __device__ __forceinline__ uint32_t magnitude(uint32_t w) { return w & 0x7fff7fffu; }
  static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) { return max_u16x2(a, b); }
  static __device__ __forceinline__ uint32_t bits(uint32_t m, int half) { return half ? m & 0xffff0000u : m << 16; }      // of fp32
};
template <> struct Eight<float> {
  static constexpr int W = 8;
  uint32_t w[8];
  __device__ __forceinline__ void load(const float* p) {
    const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  }
  __device__ __forceinline__ void set(int e, const float* p) { w[e] = __float_as_uint(*p); }
  __device__ __forceinline__ float at(int e) const { return __uint_as_float(w[e]); }
  static __device__ __forceinline__ uint32_t magnitude(uint32_t w) { return w & 0x7fffffffu; }
  static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) { return max(a, b); }
  static __device__ __forceinline__ uint32_t bits(uint32_t m, int) { return m; }
};
constexpr uint32_t kInf = 0x7f800000u;

// the largest magnitude of eight values, as bits of fp32
template <typename T> __device__ __forceinline__ uint32_t top8(const Eight<T>& x) {
  uint32_t m = Eight<T>::magnitude(x.w[0]);
#pragma unroll
  for (int i = 1; i < Eight<T>::W; i++) m = Eight<T>::most(m, Eight<T>::magnitude(x.w[i]));
  return sizeof(T) == 2 ? max(m & 0xffff0000u, m << 16) : m;
}
template <typename T> __device__ __forceinline__ uint32_t finite_top8(const Eight<T>& x) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) m = max(m, finite_bits(x.at(e)));
  return m;
}
// What is not finite becomes NaN, where a maximum said that there is any.  (Asked of every value on its way to 8 bits, it was a seventh of the quantiser's instructions.)
template <typename T> __device__ __forceinline__ void no_inf(Eight<T>& x) {
#pragma unroll
  for (int i = 0; i < Eight<T>::W; i++) {
    if (sizeof(T) == 4) { if ((x.w[i] & 0x7fffffffu) >= kInf) x.w[i] = 0x7fffffffu; }
    else {
      if ((x.w[i] & 0x7fffu) >= kInf >> 16) x.w[i] |= 0x7fffu;
      if ((x.w[i] & 0x7fff0000u) >= kInf) x.w[i] |= 0x7fff0000u;
    }
  }
}
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d, float f) {
  float x, y, z, w;
  unpack2(mul2(pack2(a, b), both2(f)), x, y);
  unpack2(mul2(pack2(c, d), both2(f)), z, w);
  return e4m3_four(x, y, z, w);
}
template <typename T> __device__ __forceinline__ uint2 pack_row(const Eight<T>& x, float f) { return make_uint2(pack4(x.at(0), x.at(1), x.at(2), x.at(3), f), pack4(x.at(4), x.at(5), x.at(6), x.at(7), f)); }

}  // namespace piccl_ops
