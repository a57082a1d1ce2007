// The products of fp8_gemm.cu for at most 64 rows, as in decoding: C[M, N] = A[M, K] B[N, K]^T + bias, bound by the bytes of B.
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

// A in shared memory: 8 T rows of kb * 128 bytes, 16-byte pieces of a block moved by the row so that eight lanes beside each other, four pieces of two rows, meet in no bank, and the scales as
// powers of two in fp32 for each block and row.
struct FewA {
  uint4* x; float* f; int kb;
  __device__ __forceinline__ uint4* piece(int row, int block, int i) const { return x + ((size_t)row * kb + block) * 8 + (i ^ (row & 1) << 2 ^ (row >> 1 & 3)); }
  __device__ __forceinline__ float* power(int row, int block, int rows) const { return f + (size_t)block * rows + row; }
};

// R: groups of 16 rows of B, T: groups of 8 rows of A, D: blocks of B that a warp has under way
template <int R, int T, int D, bool QUANT, typename O>
__global__ void __launch_bounds__(256, R * T <= 2 ? 2 : 1) fp8_few_kernel(const FewArgs a) {
  constexpr int ROWS = 16 * R, COLS = 8 * T;
  extern __shared__ __align__(16) uint4 few_smem[];
  const FewA A{few_smem, reinterpret_cast<float*>(few_smem + (size_t)COLS * a.kb * 8), a.kb};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.x * ROWS;
  const long long pitch = 128ll * a.kb;
  // B on its way into L2 while the kernel before this one ends (a hint: whatever that kernel writes is seen all the same)
  for (int i = threadIdx.x; i < ROWS * a.kb; i += 256) {
    const int row = row0 + i / a.kb;
    if (row < a.N) asm volatile("prefetch.global.L2 [%0];" ::"l"(a.w + row * pitch + (i % a.kb) * 128ll));
  }
  pdl_begin();
  struct Part { uint4 w[R][2][2]; uint32_t s[R][2]; } part[D];      // rows g and g + 8 of a group, 16 bytes of each of two chunks of 64 k; their scales
  auto load = [&](Part& p, int kb) {
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int row = row0 + 16 * r + 8 * h + g;
#pragma unroll
        for (int c = 0; c < 2; c++) p.w[r][h][c] = row < a.N ? __ldg(reinterpret_cast<const uint4*>(a.w + row * pitch + kb * 128ll + c * 64 + t * 16)) : make_uint4(0, 0, 0, 0);
        p.s[r][h] = row < a.N ? a.sw[scale_at(row, kb, a.k4)] : 1u;
      }
  };
#pragma unroll
  for (int d = 0; d < D; d++) if (warp + 8 * d < a.kb) load(part[d], warp + 8 * d);
  // A: 8 lanes to a row and block, 16 values each, U of them on their way at a time.  (Rows from M on stay what they were: they only reach sums that nobody reads.)
  {
    constexpr int U = QUANT ? 4 : 8;
    const int l8 = threadIdx.x & 7, items = a.M * a.kb, all = (items + 31) / 32 * 32;      // whole warps go round together
    for (int i0 = threadIdx.x >> 3; i0 < all; i0 += 32 * U) {
      uint32_t w[U][QUANT ? 8 : 4];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int i = i0 + 32 * u, m = i / a.kb, kb = i - m * a.kb, c = kb * 128 + l8 * 16;
#pragma unroll
        for (int e = 0; e < (QUANT ? 8 : 4); e++) w[u][e] = 0;
        if constexpr (QUANT) {
#pragma unroll
          for (int h = 0; h < 2; h++) if (i < items && c + 8 * h < a.K) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(a.x + m * a.stride + c + 8 * h));
            w[u][4 * h] = v.x; w[u][4 * h + 1] = v.y; w[u][4 * h + 2] = v.z; w[u][4 * h + 3] = v.w;
          }
        } else if (i < items) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(a.a + m * pitch + c));
          w[u][0] = v.x; w[u][1] = v.y; w[u][2] = v.z; w[u][3] = v.w;
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int i = i0 + 32 * u, m = i / a.kb, kb = i - m * a.kb;
        if (i - (threadIdx.x >> 3 & 3) >= items) break;      // none of the warp's four
        uint4 piece; uint32_t byte = 1;
        if constexpr (QUANT) {
          Eight<bf16> v[2];
#pragma unroll
          for (int e = 0; e < 4; e++) { v[0].w[e] = w[u][e]; v[1].w[e] = w[u][4 + e]; }
          uint32_t top = max(top8(v[0]), top8(v[1]));
          const bool odd = __any_sync(0xffffffffu, top >= kInf);
          if (odd) top = max(finite_top8(v[0]), finite_top8(v[1]));
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
          byte = scale_byte(top);
          const float f = scale_inverse(byte);
          const uint2 lo = pack_row(v[0], f, odd), hi = pack_row(v[1], f, odd);
          piece = make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else {
          piece = make_uint4(w[u][0], w[u][1], w[u][2], w[u][3]);
          if (l8 == 0 && i < items) byte = a.sa[scale_at(m, kb, a.k4)];
        }
        if (i < items) {
          *A.piece(m, kb, l8) = piece;
          if (l8 == 0) *A.power(m, kb, COLS) = scale_value(byte);
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
        const float2 fx = *reinterpret_cast<const float2*>(A.power(8 * n + 2 * t, kb, COLS));
#pragma unroll
        for (int r = 0; r < R; r++) {
          float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < 2; k++) {
            mma_e4m3(c, p.w[r][0][k].x, p.w[r][1][k].x, p.w[r][0][k].y, p.w[r][1][k].y, b[k].x, b[k].y);
            mma_e4m3(c, p.w[r][0][k].z, p.w[r][1][k].z, p.w[r][0][k].w, p.w[r][1][k].w, b[k].z, b[k].w);
          }
          const float f0 = scale_value(p.s[r][0]), f1 = scale_value(p.s[r][1]);
          acc[r][n][0] = fmaf(c[0] * f0, fx.x, acc[r][n][0]); acc[r][n][1] = fmaf(c[1] * f0, fx.y, acc[r][n][1]);
          acc[r][n][2] = fmaf(c[2] * f1, fx.x, acc[r][n][2]); acc[r][n][3] = fmaf(c[3] * f1, fx.y, acc[r][n][3]);
        }
      }
      if (kb + 8 * D < a.kb) load(part[d], kb + 8 * D);
    }
  }
  __syncthreads();                                         // A has been read: the sums take its place
  float* const sums = reinterpret_cast<float*>(few_smem);  // [8][COLS][ROWS + 1]
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int n = 0; n < T; n++)
#pragma unroll
      for (int i = 0; i < 4; i++) sums[(warp * COLS + 8 * n + 2 * t + (i & 1)) * (ROWS + 1) + 16 * r + 8 * (i >> 1) + g] = acc[r][n][i];
  __syncthreads();
  for (int e = threadIdx.x; e < a.M * ROWS; e += 256) {
    const int m = e / ROWS, n = e % ROWS;
    if (row0 + n >= a.N) continue;
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < 8; q++) s += sums[(q * COLS + m) * (ROWS + 1) + n];
    if (a.bias) s += __bfloat162float(a.bias[row0 + n]);
    static_cast<O*>(a.out)[(size_t)m * a.N + row0 + n] = (O)s;
  }
}

static size_t few_smem_bytes(int rows, int cols, int kb) {
  const size_t a = (size_t)cols * kb * (128 + 4), sums = (size_t)8 * cols * (rows + 1) * 4;
  return a > sums ? a : sums;
}
constexpr size_t kFewSmem = 200 * 1024;

template <int R, int T, int D, bool QUANT, typename O> static int few(const FewArgs& g, cudaStream_t s) {
  static std::atomic<bool> ready[64];
  int dev = 0; cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return -6;
  const auto fn = fp8_few_kernel<R, T, D, QUANT, O>;
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem) != cudaSuccess) return -4;
    ready[dev] = true;
  }
  return launch_pdl(fn, dim3((g.N + 16 * R - 1) / (16 * R)), 256, few_smem_bytes(16 * R, 8 * T, g.kb), s, g) == cudaSuccess ? 0 : -5;
}
template <bool QUANT, typename O> static int few(const FewArgs& g, cudaStream_t s) {
  const bool wide = g.N > 32 * 148;
  if (g.M <= 8) return wide ? few<2, 1, 2, QUANT, O>(g, s) : few<1, 1, 4, QUANT, O>(g, s);
  if (g.M <= 16) return wide ? few<2, 2, 2, QUANT, O>(g, s) : few<1, 2, 3, QUANT, O>(g, s);
  if (g.M <= 32) return few<1, 4, 3, QUANT, O>(g, s);
  return few<1, 8, 2, QUANT, O>(g, s);
}

// Whether the kernel is the one for M rows of K values: A has to fit into shared memory, and what the blocks of an SM take in of it, each for itself, has to be little beside B.  Against the quantiser
// and the pairs' kernel (us, one launch and two): M 1, N 4096, K 1024 / 4096 / 8192: 3.9 / 6.3 / 9.5 and 7.8 / 16.1 / 28.6; M 8: 4.0 / 9.2 / 15.5 and 6.8 / 13.9 / 24.8; M 16, N 1024, K 2048 / 4096: 5.9 / 10.8
// and 7.1 / 9.5; M 8, N 16384, K 1024 / 4096: 9.0 / 25.7 and 9.8 / 20.8; M 32, N 1024, K 1024 / 2048: 5.7 / 9.0 and 6.5 / 7.2.
bool fp8_few_takes(int M, int N, long long K) {
  if (M > 64 || K > 1 << 20) return false;
  const int cols = M <= 8 ? 8 : M <= 16 ? 16 : M <= 32 ? 32 : 64, kb = (int)((K + 127) / 128);
  const bool wide = N > 32 * 148 && M <= 16;
  const long long blocks = (N + (wide ? 32 : 16) - 1) / (wide ? 32 : 16), taken = (blocks + 147) / 148 * M * kb;
  return few_smem_bytes(32, cols, kb) <= kFewSmem && taken <= (M > 8 ? 256 : N > 32 * 148 ? 512 : 1024);
}
// x: A in bf16 (on 16-byte boundaries, K a multiple of 8), or null: values a with scales sa
int fp8_few(const bf16* x, long long stride, const void* a, const void* sa, const void* b, const void* sb, const void* bias, void* out, int f32, int M, int N, int K, void* stream) {
  const FewArgs g{(const uint8_t*)b, (const uint8_t*)sb, (const uint8_t*)a, (const uint8_t*)sa, x, stride, (const bf16*)bias, out, M, N, K, (K + 127) / 128, (K + 511) / 512};
  const cudaStream_t s = (cudaStream_t)stream;
  if (!fp8_few_takes(M, N, K)) return -1;
  if (x) return f32 ? few<true, float>(g, s) : few<true, bf16>(g, s);
  return f32 ? few<false, float>(g, s) : few<false, bf16>(g, s);
}

}  // namespace piccl_ops
