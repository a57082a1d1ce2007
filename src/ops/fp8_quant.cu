// bf16 or fp32 matrices -> e4m3 with a power of two for each block of 128 (fp8.cuh), along the rows, along the columns (the transposed copy, which a product
// over the other dimension takes) or both in one pass over the matrix.  Square: one power of two for each 128 x 128, so that both copies stand for the same values.
#include <atomic>
#include "fp8.cuh"

namespace piccl_ops {

struct QuantArgs {
  const void* x; long long stride;               // elements between rows
  uint8_t *q, *qs, *t, *ts;                      // rows: [R][kc], scales; transposed: [C][kr], scales
  long long R, C, kc, kr;                        // kc, kr: C and R rounded up to 128
  int c4, r4;                                    // blocks of 512 columns, rows
};

// columns [c, c + 8) of a row, zeros from C on; VEC: rows start on 16-byte boundaries and C is a multiple of 8
template <typename T, bool VEC> __device__ __forceinline__ void load8(const T* row, long long c, long long C, Eight<T>& x) {
#pragma unroll
  for (int i = 0; i < Eight<T>::W; i++) x.w[i] = 0;
  if (VEC) { if (c < C) x.load(row + c); }
  else
#pragma unroll
    for (int e = 0; e < 8; e++) if (c + e < C) x.set(e, row + c + e);
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
  Eight<T> v[2];
  load8<T, VEC>(x, c, a.C, v[0]);
  load8<T, VEC>(x, c + 8, a.C, v[1]);
  uint32_t top = max(top8(v[0]), top8(v[1]));
  if (__any_sync(0xffffffffu, top >= kInf)) { top = max(finite_top8(v[0]), finite_top8(v[1])); no_inf(v[0]); no_inf(v[1]); }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const uint32_t byte = scale_byte(top);
  const float f = scale_inverse(byte);
  if (c < a.kc) {
    const uint2 lo = pack_row(v[0], f), hi = pack_row(v[1], f);
    *reinterpret_cast<uint4*>(a.q + row * a.kc + c) = make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
  uint32_t all = byte << (8 * (lane >> 3));
  all |= __shfl_xor_sync(0xffffffffu, all, 8);
  all |= __shfl_xor_sync(0xffffffffu, all, 16);
  if (lane == 0) *word = all;
}

// A block has a tile of 128 x 128 in registers as it came, a thread 8 x 8 of it (16 lanes beside each other to a row).  The largest magnitudes of its rows and columns go through shared memory
// at one barrier; half of the threads then put the rows' together, half the columns'.  (The rows' by shuffles, 32 a thread: 42 us for
// 8192 x 4096 bf16 both ways, in place of 26.5.)  Bound by the latencies of loads and barriers at 17 instructions a value, 5.1 TB/s; four blocks to an SM, at 64 registers and a spill of 16 bytes (28 stored and 56 loaded where rows are read value by value), take 26.5 us where three take 27.2.
// Magnitudes of the two kinds: 128 lines of 16 partial maxima, a line's partial i at [i][line], and every [i] moved on by 16 bytes so that threads side by side do not meet in a bank.
template <typename T> struct Tops {
  static constexpr int PITCH = 128 * sizeof(T) + 16;       // bf16: 16 bits each
  __align__(16) uint8_t b[16 * PITCH];
  __device__ __forceinline__ uint4* eight(int i, int g) { return reinterpret_cast<uint4*>(b + i * PITCH + g * 8 * sizeof(T)); }
  // the maximum of a line, as bits of fp32
  __device__ __forceinline__ uint32_t line(int l) const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) m = max(m, sizeof(T) == 2 ? (uint32_t)*reinterpret_cast<const uint16_t*>(b + i * PITCH + 2 * l) : *reinterpret_cast<const uint32_t*>(b + i * PITCH + 4 * l));
    return sizeof(T) == 2 ? m << 16 : m;
  }
};
template <typename T, bool VEC, bool ROWS, bool COLS, bool SQUARE>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2) quant_tile_kernel(const QuantArgs a) {
  constexpr int W = Eight<T>::W, B = sizeof(T) == 2;
  union Shared {
    struct { Tops<T> rows, cols; } tops;
    uint8_t turned[COLS ? 128 * 128 : 16];
    uint32_t warps[8];
  };
  __shared__ __align__(16) Shared sh;
  __shared__ __align__(8) uint8_t row_bytes[128], col_bytes[128];
  pdl_begin();
  const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4;
  const int bx = blockIdx.x % (int)(a.kc >> 7), by = blockIdx.x / (int)(a.kc >> 7);
  const long long r0 = by * 128ll + rg * 8, c0 = bx * 128ll + cg * 8;
  Eight<T> v[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    if (r0 + i < a.R) load8<T, VEC>(static_cast<const T*>(a.x) + (r0 + i) * a.stride, c0, a.C, v[i]);
    else
#pragma unroll
      for (int e = 0; e < W; e++) v[i].w[e] = 0;
  }
  // the largest magnitudes of the thread's columns, and of all
  uint32_t col[W], top = 0;
#pragma unroll
  for (int e = 0; e < W; e++) {
    col[e] = Eight<T>::magnitude(v[0].w[e]);
#pragma unroll
    for (int i = 1; i < 8; i++) col[e] = Eight<T>::most(col[e], Eight<T>::magnitude(v[i].w[e]));
    top = max(top, B ? max(col[e] & 0xffff0000u, col[e] << 16) : col[e]);
  }
  // bytes of blocks beyond the last one, up to a whole word
  const int more_c = bx + 1 == (int)(a.kc >> 7) ? 4 * a.c4 - bx : 1, more_r = by + 1 == (int)(a.kr >> 7) ? 4 * a.r4 - by : 1;
  const int l = threadIdx.x & 127;
  const bool for_rows = threadIdx.x < 128;
  auto write_scales = [&](uint32_t byte) {                 // of line l of the rows or columns
    if (for_rows ? ROWS : COLS) {
      uint8_t* const to = for_rows ? a.qs : a.ts;
      const long long line = (for_rows ? by : bx) * 128ll + l;
      const int block = for_rows ? bx : by, more = for_rows ? more_c : more_r, four = for_rows ? a.c4 : a.r4;
      to[scale_at(line, block, four)] = byte;
      for (int k = 1; k < more; k++) to[scale_at(line, block + k, four)] = 1;
    }
  };
  float square = 0.f;
  if (SQUARE) {
    if (__syncthreads_or(top >= kInf)) {
      top = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) { top = max(top, finite_top8(v[i])); no_inf(v[i]); }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) sh.warps[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) top = max(top, sh.warps[w]);
    const uint32_t byte = scale_byte(top);
    square = scale_inverse(byte);
    write_scales((for_rows ? by * 128ll + l < a.R : bx * 128ll + l < a.C) ? byte : 1);
    if (COLS) __syncthreads();                             // the maxima have been read
  } else {
    uint32_t row[W];                                       // of the thread's rows, in pairs as the columns
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t m = top8(v[i]);
      if (B) row[i >> 1] = i & 1 ? row[i >> 1] | m : m >> 16;
      else row[i] = m;
    }
    if (__syncthreads_or(top >= kInf)) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const uint32_t m = finite_top8(v[i]);
        if (B) row[i >> 1] = i & 1 ? row[i >> 1] | m : m >> 16;
        else row[i] = m;
      }
#pragma unroll
      for (int e = 0; e < W; e++) {
        uint32_t m[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
          for (int h = 0; h < 8 / W; h++) m[h] = max(m[h], finite_bits(v[i].at(8 / W * e + h)));
        col[e] = B ? m[0] >> 16 | (m[1] & 0xffff0000u) : m[0];
      }
#pragma unroll
      for (int i = 0; i < 8; i++) no_inf(v[i]);
    }
#pragma unroll
    for (int e = 0; e < W; e += 4) {
      if (ROWS) sh.tops.rows.eight(cg, rg)[e / 4] = make_uint4(row[e], row[e + 1], row[e + 2], row[e + 3]);
      if (COLS) sh.tops.cols.eight(rg, cg)[e / 4] = make_uint4(col[e], col[e + 1], col[e + 2], col[e + 3]);
    }
    __syncthreads();
    if (for_rows ? ROWS : COLS) {
      const uint32_t byte = scale_byte((for_rows ? sh.tops.rows : sh.tops.cols).line(l));
      (for_rows ? row_bytes : col_bytes)[l] = byte;
      write_scales(byte);
    }
    __syncthreads();
  }
  if (ROWS) {
    const uint2 eight = SQUARE ? make_uint2(0, 0) : *reinterpret_cast<const uint2*>(row_bytes + rg * 8);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float f = SQUARE ? square : scale_inverse(((i < 4 ? eight.x : eight.y) >> (8 * (i & 3))) & 255u);
      if (r0 + i < a.R) *reinterpret_cast<uint2*>(a.q + (r0 + i) * a.kc + c0) = pack_row(v[i], f);
    }
  }
  if (COLS) {
    // eight rows of a column are 8 bytes of the turned tile; their place in its row of 16 is moved by the column, or 16 lanes would meet in one bank
    const uint2 eight = SQUARE ? make_uint2(0, 0) : *reinterpret_cast<const uint2*>(col_bytes + cg * 8);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float f = SQUARE ? square : scale_inverse(((e < 4 ? eight.x : eight.y) >> (8 * (e & 3))) & 255u);
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; i++) w[i] = v[i].at(e);
      *reinterpret_cast<uint2*>(sh.turned + (cg * 8 + e) * 128 + ((rg ^ cg) << 3)) = make_uint2(pack4(w[0], w[1], w[2], w[3], f), pack4(w[4], w[5], w[6], w[7], f));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int c = i * 16 + rg;
      if (bx * 128ll + c < a.C)
        *reinterpret_cast<uint2*>(a.t + (bx * 128ll + c) * a.kr + by * 128ll + cg * 8) = *reinterpret_cast<const uint2*>(sh.turned + c * 128 + ((cg ^ (c >> 3)) << 3));
    }
  }
}

// Tiles are spread evenly over the SMs: where there are fewer than fit at once, a block asks for so much shared memory that no SM takes more than its share.  (Left alone some take four and some
// none: 2331 x 2304 bf16, 342 tiles, 6.9 us with room for four blocks to an SM and 5.8 with room for three; 4096 x 1024, 256 tiles, 5.5 and, with room for two, 4.6.)
typedef void (*TileFn)(QuantArgs);
static cudaError_t launch_tiles(TileFn fn, std::atomic<bool> (&ready)[64], const QuantArgs& a, cudaStream_t s) {
  int dev = 0; cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  constexpr int ROOM[3] = {200 << 10, 90 << 10, 55 << 10};      // beside 17 KiB of its own: one, two, three blocks in an SM's 228 KiB
  if (!ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute((const void*)fn, cudaFuncAttributeMaxDynamicSharedMemorySize, ROOM[0]);
    if (e != cudaSuccess) return e;
    ready[dev] = true;
  }
  const long long tiles = a.kc / 128 * (a.kr / 128), share = (tiles + 147) / 148;
  return launch_pdl(fn, dim3((unsigned)tiles), 256, share <= 3 ? ROOM[share - 1] : 0, s, a);
}
template <typename T, bool VEC, bool ROWS, bool COLS, bool SQUARE> static cudaError_t tiles(const QuantArgs& a, cudaStream_t s) {
  static std::atomic<bool> ready[64];
  return launch_tiles(quant_tile_kernel<T, VEC, ROWS, COLS, SQUARE>, ready, a, s);
}
template <typename T, bool VEC>
static cudaError_t quantize(const QuantArgs& a, int square, cudaStream_t s) {
  if (!a.t && !square) {
    const long long warps = (a.R + 127) / 128 * 128 * a.c4;
    return launch_pdl(quant_rows_kernel<T, VEC>, dim3((unsigned)((warps + 7) / 8)), 256, 0, s, a);
  }
  if (square) return !a.t ? tiles<T, VEC, true, false, true>(a, s) : a.q ? tiles<T, VEC, true, true, true>(a, s) : tiles<T, VEC, false, true, true>(a, s);
  return a.q ? tiles<T, VEC, true, true, false>(a, s) : tiles<T, VEC, false, true, false>(a, s);
}

}  // namespace piccl_ops

using namespace piccl_ops;

extern "C" {

// x: [R, C], rows `stride` elements apart; fp32: float, else bf16.  q [R][C up to 128] with scales qs and t [C][R up to 128] with scales ts: either pair may be null, not both.
// x at any element's address; q, qs, t and ts on 16-byte boundaries.
int piccl_ops_fp8_quantize(const void* x, int fp32, long long R, long long C, long long stride, void* q, void* qs, void* t, void* ts, int square, void* stream) {
  if (R <= 0 || C <= 0 || R > 0x7fffff00ll || C > 0x7fffff00ll || stride < C) return -1;
  if (!x || (!q && !t) || !q != !qs || !t != !ts) return -2;
  const uintptr_t esz = fp32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(x) & (esz - 1)) || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(t) | reinterpret_cast<uintptr_t>(qs) | reinterpret_cast<uintptr_t>(ts)) & 15)) return -2;
  QuantArgs a{x, stride, (uint8_t*)q, (uint8_t*)qs, (uint8_t*)t, (uint8_t*)ts, R, C, (C + 127) / 128 * 128, (R + 127) / 128 * 128, (int)((C + 511) / 512), (int)((R + 511) / 512)};
  if ((a.kr / 128) * (a.kc / 128) > 0x7fffffffll || a.kr * a.c4 / 8 > 0x7ffffff0ll) return -1;      // blocks of a grid
  const bool vec = C % 8 == 0 && stride * esz % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  const cudaStream_t s = (cudaStream_t)stream;
  const cudaError_t e = fp32 ? (vec ? quantize<float, true>(a, square, s) : quantize<float, false>(a, square, s)) : (vec ? quantize<bf16, true>(a, square, s) : quantize<bf16, false>(a, square, s));
  return e == cudaSuccess ? 0 : (int)e;
}

}  // extern "C"
