// The products of fp8_gemm.cu for at most 32 rows, as in decoding: C[M, N] = A[M, K] B[N, K]^T + bias, bound by the bytes of B.
//
// A block has 16 or 32 rows of B, its eight warps take the k-blocks of 128 in turn: a warp reads its part of B straight into the fragments of mma.sync (B's rows are the fragment's 16 rows, A's
// rows its 8 columns; k may stand in any order that both sides share, so a lane's 16 bytes are contiguous), sums a block of 128 and adds it to its sums in fp32, scaled by the two powers of two.  The
// warps' sums meet in shared memory and are added in the warps' order.  No part of B is staged and nothing waits for another block; a warp has several blocks of B under way while all warps
// bring A into shared memory.  (Tensor cores that need descriptors, TMEM and barriers have nothing to gain where 2 KiB a warp and block are read once.)
// A may come as bf16: it is rounded on its way into shared memory, which saves the launch, and the scratch, of a quantiser; every block reads all of A for it.
#include <atomic>
#include "fp8.cuh"

namespace piccl_ops {

struct FewArgs {
  const uint8_t *w, *sw, *a, *sa;    // B's values and scales, A's
  const bf16* x; long long stride;   // or A itself
  const bf16* bias; void* out;
  int M, N, K, kb, k4;
};

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// acc += what a block of 128 k gives: rows g and g + 8 of 16 rows of B (two chunks of 64 k, 16 bytes each), row g of 8 rows of A; f: bytes of the scales of the rows of B, x: of rows 2 t and 2 t + 1 of A, all moved to bit 22.
// The product of two scales has twice the range of fp32, and one may be far above 1 where the other is far below, so half of their sum of exponents is multiplied by first, the rest after it: each partial
// result is then between 2^-145 and the last one.
__device__ __forceinline__ void add_block(float (&acc)[4], const uint4 (&w)[2][2], const uint4 (&b)[2], uint32_t f0, uint32_t f1, uint32_t x0, uint32_t x1) {
  float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 2; k++) {
    mma_e4m3(c, w[0][k].x, w[1][k].x, w[0][k].y, w[1][k].y, b[k].x, b[k].y);
    mma_e4m3(c, w[0][k].z, w[1][k].z, w[0][k].w, w[1][k].w, b[k].z, b[k].w);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t both = (i < 2 ? f0 : f1) + (i & 1 ? x1 : x0), half = both & 0x7f800000u;
    acc[i] = fmaf(c[i] * __uint_as_float(half), __uint_as_float(2 * both - half), acc[i]);
  }
}
// sums: [8 warps][8 T][16 R + 1]
template <int R, int T> __device__ __forceinline__ void put_sums(float* sums, const float (&acc)[R][T][4], int warp, int g, int t) {
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int n = 0; n < T; n++)
#pragma unroll
      for (int i = 0; i < 4; i++) sums[(warp * 8 * T + 8 * n + 2 * t + (i & 1)) * (16 * R + 1) + 16 * r + 8 * (i >> 1) + g] = acc[r][n][i];
}
template <int R, int T, typename O> __device__ __forceinline__ void write_sums(const FewArgs& a, const float* sums, int row0) {
  constexpr int ROWS = 16 * R;
  for (int e = threadIdx.x; e < a.M * ROWS; e += 256) {
    const int m = e / ROWS, n = e % ROWS;
    if (row0 + n >= a.N) continue;
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < 8; q++) s += sums[(q * 8 * T + m) * (ROWS + 1) + n];
    if (a.bias) s += __bfloat162float(a.bias[row0 + n]);
    static_cast<O*>(a.out)[(size_t)m * a.N + row0 + n] = (O)s;
  }
}
// A block's rows of B on their way into L2 while the kernel before this one ends (a hint: whatever that kernel writes is seen all the same)
__device__ __forceinline__ void prefetch_rows(const FewArgs& a, int row0, int rows) {
  for (int i = threadIdx.x; i < rows * a.kb; i += 256) {
    const int row = row0 + i / a.kb;
    if (row < a.N) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.w + (row * (long long)a.kb + i % a.kb) * 128));
  }
}

// A in shared memory: 8 T rows of kb * 128 bytes, 16-byte pieces of a block moved by the row so that eight lanes beside each other, four pieces of two rows, meet in no bank, and the scales'
// bytes, moved to bit 22, for each block and row.
struct FewA {
  uint4* x; uint32_t* f; int kb;
  __device__ __forceinline__ uint4* piece(int row, int block, int i) const { return x + ((size_t)row * kb + block) * 8 + (i ^ (row & 1) << 2 ^ (row >> 1 & 3)); }
  __device__ __forceinline__ uint32_t* scale(int row, int block, int rows) const { return f + (size_t)block * rows + row; }
};

// R: groups of 16 rows of B, T: groups of 8 rows of A, D: blocks of B that a warp has under way
template <int R, int T, int D, typename O>
__global__ void __launch_bounds__(256, R * T <= 2 ? 2 : 1) fp8_few_kernel(const FewArgs a) {
  constexpr int ROWS = 16 * R, COLS = 8 * T;
  extern __shared__ __align__(16) uint4 few_smem[];
  const FewA A{few_smem, reinterpret_cast<uint32_t*>(few_smem + (size_t)COLS * a.kb * 8), a.kb};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.x * ROWS;
  const long long pitch = 128ll * a.kb;
  prefetch_rows(a, row0, ROWS);
  pdl_begin();
  struct Part { uint4 w[R][2][2]; uint32_t s[R][2]; } part[D];      // rows g and g + 8 of a group, 16 bytes of each of two chunks of 64 k; their scales
  auto load = [&](Part& p, int kb) {
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int row = row0 + 16 * r + 8 * h + g;
#pragma unroll
        for (int c = 0; c < 2; c++) p.w[r][h][c] = row < a.N ? *reinterpret_cast<const uint4*>(a.w + row * pitch + kb * 128ll + c * 64 + t * 16) : make_uint4(0, 0, 0, 0);
        p.s[r][h] = row < a.N ? a.sw[scale_at(row, kb, a.k4)] : 1u;
      }
  };
#pragma unroll
  for (int d = 0; d < D; d++) if (warp + 8 * d < a.kb) load(part[d], warp + 8 * d);
  // A: 8 lanes to a row and block, 16 values each, U of them on their way at a time.  (Rows from M on stay what they were: they only reach sums that nobody reads.)
  {
    constexpr int U = 4;
    const int l8 = threadIdx.x & 7, items = a.M * a.kb, all = (items + 31) / 32 * 32;      // whole warps go round together
    for (int i0 = threadIdx.x >> 3; i0 < all; i0 += 32 * U) {
      Eight<bf16> v[U][2];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int i = i0 + 32 * u, m = i / a.kb, c = (i - m * a.kb) * 128 + l8 * 16;
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
          for (int e = 0; e < 4; e++) v[u][h].w[e] = 0;
          if (i < items && c + 8 * h < a.K) v[u][h].load(a.x + m * a.stride + c + 8 * h);
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int i = i0 + 32 * u, m = i / a.kb, kb = i - m * a.kb;
        if (i - (threadIdx.x >> 3 & 3) >= items) break;      // none of the warp's four
        uint32_t top = max(top8(v[u][0]), top8(v[u][1]));
        if (__any_sync(0xffffffffu, top >= kInf)) { top = max(finite_top8(v[u][0]), finite_top8(v[u][1])); no_inf(v[u][0]); no_inf(v[u][1]); }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const uint32_t byte = scale_byte(top);
        const float f = scale_inverse(byte);
        const uint2 lo = pack_row(v[u][0], f), hi = pack_row(v[u][1], f);
        if (i < items) {
          *A.piece(m, kb, l8) = make_uint4(lo.x, lo.y, hi.x, hi.y);
          if (l8 == 0) *A.scale(m, kb, COLS) = byte << 22;
        }
      }
    }
  }
  __syncthreads();
  float acc[R][T][4];
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int n = 0; n < T; n++)
#pragma unroll
      for (int i = 0; i < 4; i++) acc[r][n][i] = 0.f;
  for (int base = warp; base < a.kb; base += 8 * D) {
#pragma unroll
    for (int d = 0; d < D; d++) {
      const int kb = base + 8 * d;
      if (kb >= a.kb) break;
      const Part& p = part[d];
#pragma unroll
      for (int n = 0; n < T; n++) {
        uint4 b[2];                                        // row 8 n + g of A
#pragma unroll
        for (int k = 0; k < 2; k++) b[k] = *A.piece(8 * n + g, kb, 4 * k + t);
        const uint2 fx = *reinterpret_cast<const uint2*>(A.scale(8 * n + 2 * t, kb, COLS));
#pragma unroll
        for (int r = 0; r < R; r++) add_block(acc[r][n], p.w[r], b, p.s[r][0] << 22, p.s[r][1] << 22, fx.x, fx.y);
      }
      if (kb + 8 * D < a.kb) load(part[d], kb + 8 * D);
    }
  }
  __syncthreads();                                         // A has been read: the sums take its place
  float* const sums = reinterpret_cast<float*>(few_smem);
  put_sums<R, T>(sums, acc, warp, g, t);
  __syncthreads();
  write_sums<R, T, O>(a, sums, row0);
}

// The same for A in 8 bits, read by each warp as the fragments that it needs, beside B's.
template <int R, int T, int D, typename O>
__global__ void __launch_bounds__(256, 1) fp8_fragments_kernel(const FewArgs a) {
  constexpr int ROWS = 16 * R, COLS = 8 * T;
  __shared__ float sums[8][COLS][ROWS + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.x * ROWS;
  const long long pitch = 128ll * a.kb;
  prefetch_rows(a, row0, ROWS);
  pdl_begin();
  struct Part { uint4 w[R][2][2], b[T][2]; uint32_t s[R][2], f[T][2]; } part[D];
  auto load = [&](Part& p, int kb) {
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int row = row0 + 16 * r + 8 * h + g;
#pragma unroll
        for (int c = 0; c < 2; c++) p.w[r][h][c] = row < a.N ? *reinterpret_cast<const uint4*>(a.w + row * pitch + kb * 128ll + c * 64 + t * 16) : make_uint4(0, 0, 0, 0);
        p.s[r][h] = row < a.N ? a.sw[scale_at(row, kb, a.k4)] : 1u;
      }
#pragma unroll
    for (int n = 0; n < T; n++) {
      const int m = 8 * n + g;
#pragma unroll
      for (int c = 0; c < 2; c++) p.b[n][c] = m < a.M ? *reinterpret_cast<const uint4*>(a.a + m * pitch + kb * 128ll + c * 64 + t * 16) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 2; j++) p.f[n][j] = a.sa[scale_at(8 * n + 2 * t + j, kb, a.k4)];      // (scales have room for 128 rows)
    }
  };
#pragma unroll
  for (int d = 0; d < D; d++) if (warp + 8 * d < a.kb) load(part[d], warp + 8 * d);
  float acc[R][T][4];
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int n = 0; n < T; n++)
#pragma unroll
      for (int i = 0; i < 4; i++) acc[r][n][i] = 0.f;
  for (int base = warp; base < a.kb; base += 8 * D) {
#pragma unroll
    for (int d = 0; d < D; d++) {
      const int kb = base + 8 * d;
      if (kb >= a.kb) break;
      const Part& p = part[d];
#pragma unroll
      for (int n = 0; n < T; n++)
#pragma unroll
        for (int r = 0; r < R; r++) add_block(acc[r][n], p.w[r], p.b[n], p.s[r][0] << 22, p.s[r][1] << 22, p.f[n][0] << 22, p.f[n][1] << 22);
      if (kb + 8 * D < a.kb) load(part[d], kb + 8 * D);
    }
  }
  put_sums<R, T>(&sums[0][0][0], acc, warp, g, t);
  __syncthreads();
  write_sums<R, T, O>(a, &sums[0][0][0], row0);
}

static size_t few_smem_bytes(int rows, int cols, int kb) {
  const size_t a = (size_t)cols * kb * (128 + 4), sums = (size_t)8 * cols * (rows + 1) * 4;
  return a > sums ? a : sums;
}
constexpr size_t kFewSmem = 200 * 1024;

template <int R, int T, int D, typename O> static int few_rounding(const FewArgs& g, cudaStream_t s) {
  static std::atomic<bool> ready[64];
  int dev = 0; cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return -6;
  const auto fn = fp8_few_kernel<R, T, D, O>;
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem) != cudaSuccess) return -4;
    ready[dev] = true;
  }
  return launch_pdl(fn, dim3((g.N + 16 * R - 1) / (16 * R)), 256, few_smem_bytes(16 * R, 8 * T, g.kb), s, g) == cudaSuccess ? 0 : -5;
}
template <int T, int D, typename O> static int few_fragments(const FewArgs& g, cudaStream_t s) {
  return launch_pdl(fp8_fragments_kernel<1, T, D, O>, dim3((g.N + 15) / 16), 256, 0, s, g) == cudaSuccess ? 0 : -5;
}
static bool few_wide(int N) { return N > 32 * 148; }
template <typename O> static int few(const FewArgs& g, cudaStream_t s) {
  if (g.x) {
    if (g.M <= 8) return few_wide(g.N) ? few_rounding<2, 1, 2, O>(g, s) : few_rounding<1, 1, 4, O>(g, s);
    return few_rounding<1, 2, 3, O>(g, s);
  }
  if (g.M <= 8) return few_fragments<1, 4, O>(g, s);
  if (g.M <= 16) return few_fragments<2, 3, O>(g, s);
  if (g.M <= 24) return few_fragments<3, 2, O>(g, s);
  return few_fragments<4, 1, O>(g, s);
}

// Whether these kernels are the ones for M rows: every block takes in all of A, so what counts is that and how many blocks an SM has one after the other.  us, rounding in the kernel / quantiser and
// fragments / quantiser and the pairs' kernel:
//   N 1024   K 2048  M 2 3.9 / 5.6 / 6.9, M 8 3.9 / 5.6 / 7.0, M 16 5.9 / 5.6 / 7.0    K 4096  M 2 4.2 / 5.6 / 9.4, M 8 6.4 / 5.6 / 9.4, M 32 - / 8.2 / 9.6    K 8192  M 2 6.7 / 6.7 / 14.4, M 32 - / 13.3 / 14.5
//   N 4096   K 1024  M 8 3.9 / 5.6 / 6.5, M 16 5.3 / 5.8 / 6.5, M 24 - / 6.3 / 6.5     K 4096  M 2 6.6 / 8.7 / 10.9, M 8 9.3 / 9.2 / 10.4, M 24 - / 12.4 / 10.8   K 8192  M 8 15.8 / 14.4 / 16.5, M 16 - / 16.8 / 15.4
//   N 16384  K 1024  M 2 8.4 / 10.3 / 10.5, M 8 9.4 / 10.6 / 9.7, M 16 12.2 / 12.2 / 9.5   K 4096  M 2 21.1 / 23.7 / 21.3, M 8 24.1 / 24.1 / 21.7
bool fp8_few_takes(int M, int N, long long K, bool rounded) {
  if (M > 32 || K > 1 << 20) return false;
  const bool wide = few_wide(N);
  const int kb = (int)((K + 127) / 128), rows = wide ? 32 : 16;
  const long long turns = ((N + rows - 1) / rows + 147) / 148, taken = turns * M * kb;
  if (rounded) return !wide && (turns == 1 || M <= 8 || taken <= (M <= 16 ? 1024 : 512));
  return M <= 16 && !(wide && M > 8) && few_smem_bytes(rows, M <= 8 ? 8 : 16, kb) <= kFewSmem && taken <= (turns == 1 ? 128 : M <= 4 ? 512 : 256);
}
// x: A in bf16 (on 16-byte boundaries, K a multiple of 8), or null: values a with scales sa
int fp8_few(const bf16* x, long long stride, const void* a, const void* sa, const void* b, const void* sb, const void* bias, void* out, int f32, int M, int N, int K, void* stream) {
  const FewArgs g{(const uint8_t*)b, (const uint8_t*)sb, (const uint8_t*)a, (const uint8_t*)sa, x, stride, (const bf16*)bias, out, M, N, K, (K + 127) / 128, (K + 511) / 512};
  if (!fp8_few_takes(M, N, K, x == nullptr)) return -1;
  return f32 ? few<float>(g, (cudaStream_t)stream) : few<bf16>(g, (cudaStream_t)stream);
}

}  // namespace piccl_ops
