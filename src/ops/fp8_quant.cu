// bf16 or fp32 matrices -> e4m3 with a power of two for each block of 128 (fp8.cuh), along the rows, along the columns (the transposed copy, which a product
// over the other dimension takes) or both in one pass over the matrix.  Square: one power of two for each 128 x 128, so that both copies stand for the same values.
#include "fp8.cuh"

namespace piccl_ops {

struct QuantArgs {
  const void* x; long long stride;               // elements between rows
  uint8_t *q, *qs, *t, *ts;                      // rows: [R][kc], scales; transposed: [C][kr], scales
  long long R, C, kc, kr;                        // kc, kr: C and R rounded up to 128
  int c4, r4;                                    // blocks of 512 columns, rows
};

template <typename T> struct Loads;
template <> struct Loads<bf16> {
  static __device__ __forceinline__ void eight(const bf16* p, float (&v)[8]) { unpack8(*reinterpret_cast<const bf16x8*>(p), v); }
  static __device__ __forceinline__ float one(const bf16* p) { return __bfloat162float(*p); }
};
template <> struct Loads<float> {
  static __device__ __forceinline__ void eight(const float* p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
};
// columns [c, c + 8) of a row, zeros from C on; VEC: rows start on 16-byte boundaries and C is a multiple of 8
template <typename T, bool VEC> __device__ __forceinline__ void load8(const T* row, long long c, long long C, float (&v)[8]) {
  if (VEC) {
    if (c < C) Loads<T>::eight(row + c, v);
    else
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = 0.f;
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = c + e < C ? Loads<T>::one(row + c + e) : 0.f;
  }
}
__device__ __forceinline__ float scaled(float x, float f) { const float y = x * f; return finite_bits(x) | (x == 0.f) ? y : __uint_as_float(0x7fffffffu); }
__device__ __forceinline__ uint2 pack_e4m3(const float (&v)[8], float f) {
  uint2 o;
  o.x = e4m3_pair(scaled(v[0], f), scaled(v[1], f)) | e4m3_pair(scaled(v[2], f), scaled(v[3], f)) << 16;
  o.y = e4m3_pair(scaled(v[4], f), scaled(v[5], f)) | e4m3_pair(scaled(v[6], f), scaled(v[7], f)) << 16;
  return o;
}

// Along the rows: a warp has a row and 512 columns, a lane 16 of them, so that the four bytes of scales are one word.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quant_rows_kernel(const QuantArgs a) {
  pdl_begin();
  const int lane = threadIdx.x & 31;
  const long long item = blockIdx.x * 8ll + (threadIdx.x >> 5), row = item / a.c4;
  const int c4 = (int)(item - row * a.c4);
  if (row >= (a.R + 127) / 128 * 128) return;
  uint32_t* const word = reinterpret_cast<uint32_t*>(a.qs + scale_at(row, 4 * c4, a.c4));
  if (row >= a.R) { if (lane == 0) *word = 0x01010101u; return; }
  const T* const x = static_cast<const T*>(a.x) + row * a.stride;
  const long long c = c4 * 512ll + lane * 16;
  float v[2][8];
  load8<T, VEC>(x, c, a.C, v[0]);
  load8<T, VEC>(x, c + 8, a.C, v[1]);
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) top = max(top, max(finite_bits(v[0][e]), finite_bits(v[1][e])));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const uint32_t byte = scale_byte(top);
  const float f = scale_inverse(byte);
  if (c < a.kc) {
    const uint2 lo = pack_e4m3(v[0], f), hi = pack_e4m3(v[1], f);
    *reinterpret_cast<uint4*>(a.q + row * a.kc + c) = make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
  uint32_t all = byte << (8 * (lane >> 3));
  all |= __shfl_xor_sync(0xffffffffu, all, 8);
  all |= __shfl_xor_sync(0xffffffffu, all, 16);
  if (lane == 0) *word = all;
}

// A block has a tile of 128 x 128 in registers, a thread 8 x 8 of it (16 lanes beside each other to a row).
template <typename T, bool VEC, bool ROWS, bool COLS, bool SQUARE>
__global__ void __launch_bounds__(256) quant_tile_kernel(const QuantArgs a) {
  __shared__ uint32_t tops[16][128];
  __shared__ __align__(16) uint8_t turned[128 * 128];
  __shared__ uint8_t bytes[128];
  pdl_begin();
  const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4;
  const long long r0 = blockIdx.y * 128ll + rg * 8, c0 = blockIdx.x * 128ll + cg * 8;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    if (r0 + i < a.R) load8<T, VEC>(static_cast<const T*>(a.x) + (r0 + i) * a.stride, c0, a.C, v[i]);
    else
#pragma unroll
      for (int e = 0; e < 8; e++) v[i][e] = 0.f;
  }
  const int bx = blockIdx.x, by = blockIdx.y;
  // bytes of blocks beyond the last one, up to a whole word
  const int more_c = bx + 1 == (int)gridDim.x ? 4 * a.c4 - bx : 1, more_r = by + 1 == (int)gridDim.y ? 4 * a.r4 - by : 1;
  float square = 0.f;
  if (SQUARE) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) top = max(top, finite_bits(v[i][e]));
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[0][threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) top = max(top, tops[0][w]);
    const uint32_t byte = scale_byte(top);
    square = scale_inverse(byte);
    if (threadIdx.x < 128) {
      if (ROWS) for (int k = 0; k < more_c; k++) a.qs[scale_at(by * 128ll + threadIdx.x, bx + k, a.c4)] = k || by * 128ll + threadIdx.x >= a.R ? 1 : byte;
      if (COLS) for (int k = 0; k < more_r; k++) a.ts[scale_at(bx * 128ll + threadIdx.x, by + k, a.r4)] = k || bx * 128ll + threadIdx.x >= a.C ? 1 : byte;
    }
  }
  if (ROWS) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      float f = square;
      if (!SQUARE) {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) top = max(top, finite_bits(v[i][e]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const uint32_t byte = scale_byte(top);
        f = scale_inverse(byte);
        if (cg == 0) for (int k = 0; k < more_c; k++) a.qs[scale_at(r0 + i, bx + k, a.c4)] = k ? 1 : byte;
      }
      if (r0 + i < a.R) *reinterpret_cast<uint2*>(a.q + (r0 + i) * a.kc + c0) = pack_e4m3(v[i], f);
    }
  }
  if (COLS) {
    if (!SQUARE) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) top = max(top, finite_bits(v[i][e]));
        tops[rg][cg * 8 + e] = top;
      }
      __syncthreads();
      if (threadIdx.x < 128) {
        uint32_t top = 0;
#pragma unroll
        for (int g = 0; g < 16; g++) top = max(top, tops[g][threadIdx.x]);
        const uint32_t byte = scale_byte(top);
        bytes[threadIdx.x] = byte;
        for (int k = 0; k < more_r; k++) a.ts[scale_at(bx * 128ll + threadIdx.x, by + k, a.r4)] = k ? 1 : byte;
      }
      __syncthreads();
    }
    // eight rows of a column are 8 bytes of the turned tile; their place in its row of 16 is moved by the column, or 16 lanes would meet in one bank
#pragma unroll
    for (int e = 0; e < 8; e++) {
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; i++) w[i] = v[i][e];
      const float f = SQUARE ? square : scale_inverse(bytes[cg * 8 + e]);
      *reinterpret_cast<uint2*>(turned + (cg * 8 + e) * 128 + ((rg ^ cg) << 3)) = pack_e4m3(w, f);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int col = i * 16 + rg;
      if (bx * 128ll + col < a.C)
        *reinterpret_cast<uint2*>(a.t + (bx * 128ll + col) * a.kr + by * 128ll + cg * 8) = *reinterpret_cast<const uint2*>(turned + col * 128 + ((cg ^ (col >> 3)) << 3));
    }
  }
}

template <typename T, bool VEC>
static cudaError_t quantize(const QuantArgs& a, int square, cudaStream_t s) {
  if (!a.t && !square) {
    const long long warps = (a.R + 127) / 128 * 128 * a.c4;
    return launch_pdl(quant_rows_kernel<T, VEC>, dim3((unsigned)((warps + 7) / 8)), 256, 0, s, a);
  }
  const dim3 grid((unsigned)(a.kc / 128), (unsigned)(a.kr / 128));
  if (square) return launch_pdl(a.t ? (a.q ? quant_tile_kernel<T, VEC, true, true, true> : quant_tile_kernel<T, VEC, false, true, true>) : quant_tile_kernel<T, VEC, true, false, true>, grid, 256, 0, s, a);
  return launch_pdl(a.q ? quant_tile_kernel<T, VEC, true, true, false> : quant_tile_kernel<T, VEC, false, true, false>, grid, 256, 0, s, a);
}

}  // namespace piccl_ops

using namespace piccl_ops;

extern "C" {

// x: [R, C], rows `stride` elements apart; fp32: float, else bf16.  q [R][C up to 128] with scales qs and t [C][R up to 128] with scales ts: either pair may be null, not both.
// q, t: 8-byte aligned or better; qs, ts: 4-byte aligned.
int piccl_ops_fp8_quantize(const void* x, int fp32, long long R, long long C, long long stride, void* q, void* qs, void* t, void* ts, int square, void* stream) {
  if (R <= 0 || C <= 0 || R > 0x7fffff00ll || C > 0x7fffff00ll || stride < C) return -1;
  if (!x || (!q && !t) || !q != !qs || !t != !ts) return -2;
  const uintptr_t esz = fp32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(x) & (esz - 1)) || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(t) | reinterpret_cast<uintptr_t>(qs) | reinterpret_cast<uintptr_t>(ts)) & 15)) return -2;
  QuantArgs a{x, stride, (uint8_t*)q, (uint8_t*)qs, (uint8_t*)t, (uint8_t*)ts, R, C, (C + 127) / 128 * 128, (R + 127) / 128 * 128, (int)((C + 511) / 512), (int)((R + 511) / 512)};
  if (a.kr / 128 > 65535 && (t || square)) return -1;                     // rows of tiles of a grid
  if (a.kr * a.c4 / 8 > 0x7fffffffll) return -1;
  const bool vec = C % 8 == 0 && stride * esz % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  const cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = fp32 ? (vec ? quantize<float, true>(a, square, s) : quantize<float, false>(a, square, s)) : (vec ? quantize<bf16, true>(a, square, s) : quantize<bf16, false>(a, square, s));
  return e == cudaSuccess ? 0 : (int)e;
}

}  // extern "C"
