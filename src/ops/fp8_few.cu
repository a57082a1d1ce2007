// The products of fp8_gemm.cu for at most 64 rows, as in decoding: C[M, N] = A[M, K] B[N, K]^T + bias, bound by the bytes of B.
//
// The operands change places: a CTA has 128 rows of B as the rows of its tile and all M rows of A as its columns (16, 32 or 64), so no part of the instruction works on rows that are not
// there.  K is split over the CTAs of a cluster until the chip has a CTA or two per SM; each leaves its partial sums in shared memory, and every CTA adds a share of them up, in the order
// of the ranks, through distributed shared memory.  A may come as bf16: eight warps round it on its way into shared memory (a block of 128 each), which saves the launch, and the
// scratch, of a quantiser.
#include <cstring>
#include <mutex>
#include "../include/sm100_gemm_pair.cuh"
#include "fp8.cuh"
#include "fp8_mma.cuh"

namespace piccl_ops {

using namespace sm100;

struct FewArgs {
  CUtensorMap tw, sw, tx, sx;        // B's values and scales, A's
  const bf16* x; long long stride;   // or A itself
  const bf16* bias; void* out;
  int M, N, K, kb, k4, splits;
  int* status;
};
constexpr int FEW_THREADS = 320;

template <int T>
struct FewSmem {
  static constexpr int STAGES = T <= 32 ? 5 : 4, W_BYTES = 128 * 128, X_BYTES = T * 128, STAGE = W_BYTES + X_BYTES;
  static constexpr int SF_OFF = STAGES * STAGE, BAR_OFF = SF_OFF + STAGES * 1024, TOTAL = BAR_OFF + (2 * STAGES + 1) * 8 + 8, DYNAMIC = TOTAL + 1024;
  static_assert(128 * T * 4 <= STAGES * STAGE && 2 * (DYNAMIC + 2048) <= 228 * 1024, "partial sums lie over the ring; two CTAs to an SM");
};

__device__ __forceinline__ float cluster_load(const float* p, uint32_t rank) {
  uint32_t a; float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}

template <int T, bool QUANT, typename O>
__global__ void __launch_bounds__(FEW_THREADS) fp8_few_kernel(const __grid_constant__ FewArgs a) {
  typedef FewSmem<T> L;
  constexpr int STAGES = L::STAGES;
  constexpr uint32_t COLS = T == 16 ? 32 : T == 32 ? 64 : 128;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ int s_abort;
  __shared__ uint32_t s_tmem;
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t *const empty = full + STAGES, *const done = empty + STAGES;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = blockIdx.x % a.splits, tile = blockIdx.x / a.splits, kb0 = (int)((long long)a.kb * rank / a.splits), kb1 = (int)((long long)a.kb * (rank + 1) / a.splits);
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int s = 0; s < STAGES; s++) { mbar_init(&full[s], QUANT ? 2 : 1); mbar_init(&empty[s], 1); }
    mbar_init(done, 1);
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc_cta(&s_tmem, COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  pdl_begin();
  bool ok = true;

  if (warp == 0) {
    const bool issuer = elect_one();
    for (int kb = kb0; kb < kb1; kb++) {
      const int j = kb - kb0, st = j % STAGES;
      if (!mbar_wait(&empty[st], ((j / STAGES) & 1) ^ 1, &s_abort, kPairWaitLimitNs)) { ok = false; break; }
      uint8_t *const pw = smem + st * L::STAGE, *const ps = smem + L::SF_OFF + st * 1024;
      if (issuer) {
        const bool scales = kb == kb0 || (kb & 3) == 0;
        mbar_arrive_expect_tx(&full[st], L::W_BYTES + (QUANT ? 0 : L::X_BYTES) + (scales ? (QUANT ? 512 : 1024) : 0));
        tma_load_2d(pw, &a.tw, kb * 128, tile * 128, &full[st]);
        if (!QUANT) tma_load_2d(pw + L::W_BYTES, &a.tx, kb * 128, 0, &full[st]);
        if (scales) {
          tma_load_2d(ps, &a.sw, 0, tile * a.k4 + (kb >> 2), &full[st]);
          if (!QUANT) tma_load_2d(ps + 512, &a.sx, 0, kb >> 2, &full[st]);
        }
      }
      __syncwarp();
    }
  } else if (warp == 1) {
    const bool issuer = elect_one();
    constexpr uint32_t idesc = make_idesc_mxf8(128, T);
    const uint64_t dw0 = make_smem_desc_k128(smem), dx0 = make_smem_desc_k128(smem + L::W_BYTES), ds0 = make_smem_desc_scales(smem + L::SF_OFF);
    for (int kb = kb0; kb < kb1; kb++) {
      const int j = kb - kb0, st = j % STAGES;
      if (!mbar_wait(&full[st], (j / STAGES) & 1, &s_abort, kPairWaitLimitNs)) { ok = false; break; }
      tc_fence_after();
      const uint64_t dw = desc_advance(dw0, st * L::STAGE), dx = desc_advance(dx0, st * L::STAGE), ds = desc_advance(ds0, st * 1024);
      if (issuer) {
        const bool scales = kb == kb0 || (kb & 3) == 0;
        if (scales) scales_to_tmem(tmem + T, ds);
        if (QUANT || scales) scales_to_tmem(tmem + T + 4, desc_advance(ds, 512));
        const uint32_t byte = kb & 3;
#pragma unroll
        for (int k = 0; k < 4; k++) umma_mxf8(tmem, desc_advance(dw, k * 32), desc_advance(dx, k * 32), idesc | idesc_bytes(byte, QUANT ? 0 : byte), tmem + T, tmem + T + 4, j != 0 || k != 0);
        umma_commit_cta(&empty[st]);
      }
      __syncwarp();
    }
    if (ok && issuer) umma_commit_cta(done);
    __syncwarp();
  } else if (QUANT) {
    // a warp has every eighth block of the slice: 8 lanes to a row, 16 values each
    const int sub = lane >> 3, l8 = lane & 7;
    for (int kb = kb0 + warp - 2; kb < kb1 && ok; kb += 8) {
      const int j = kb - kb0, st = j % STAGES;
      uint8_t *const px = smem + st * L::STAGE + L::W_BYTES, *const ps = smem + L::SF_OFF + st * 1024 + 512;
      const int c = kb * 128 + l8 * 16;
      bool waited = false;
#pragma unroll 1
      for (int r0 = 0; r0 < T && r0 < a.M; r0 += 16) {
        Eight<bf16> v[4][2];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[i][h].w[e] = 0;
            if (r0 + 4 * i + sub < a.M && c + 8 * h < a.K) v[i][h].load(a.x + (r0 + 4 * i + sub) * a.stride + c + 8 * h);
          }
        if (!waited) { ok = mbar_wait(&empty[st], ((j / STAGES) & 1) ^ 1, &s_abort, kPairWaitLimitNs); waited = true; if (!ok) break; }
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int r = r0 + 4 * i + sub;
          uint32_t top = max(top8(v[i][0]), top8(v[i][1]));
          const bool odd = __any_sync(0xffffffffu, top >= kInf);
          if (odd) top = max(finite_top8(v[i][0]), finite_top8(v[i][1]));
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
          const uint32_t byte = scale_byte(top);
          const float f = scale_inverse(byte);
          const uint2 lo = pack_row(v[i][0], f, odd), hi = pack_row(v[i][1], f, odd);
          if (r < a.M) {
            *reinterpret_cast<uint4*>(px + r * 128 + ((l8 ^ (r & 7)) << 4)) = make_uint4(lo.x, lo.y, hi.x, hi.y);
            if (l8 == 0) *reinterpret_cast<uint32_t*>(ps + (r & 31) * 16 + (r >> 5) * 4) = byte;
          }
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(&full[st]);
    }
  }
  // partial sums, over the ring: all of it has been read
  float* const part = reinterpret_cast<float*>(smem);
  if (warp >= 2 && warp < 6 && ok) {
    ok = mbar_wait(done, 0, &s_abort, kPairWaitLimitNs);
    tc_fence_after();
    if (ok) {
      const int quarter = warp & 3;
#pragma unroll
      for (int q = 0; q < T / 16; q++) {
        uint32_t r[16];
        tmem_ld_32x16(tmem + ((uint32_t)(quarter * 32) << 16) + 16 * q, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; i++) if (16 * q + i < a.M) part[(16 * q + i) * 128 + quarter * 32 + lane] = __uint_as_float(r[i]);
      }
    }
  }
  if (!ok) { *(volatile int*)&s_abort = 1; if (lane == 0) atomicExch(a.status, 20 + warp); }
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();
  const int total = a.M * 128, share = (total + a.splits - 1) / a.splits, end = min(total, share * (rank + 1));
  for (int e = share * rank + threadIdx.x; e < end; e += FEW_THREADS) {
    const int n = tile * 128 + (e & 127);
    float s = 0.f;
    for (int p = 0; p < a.splits; p += 4) {
      float v[4];
#pragma unroll
      for (int q = 0; q < 4; q++) v[q] = p + q < a.splits ? cluster_load(part + e, p + q) : 0.f;
#pragma unroll
      for (int q = 0; q < 4; q++) s += v[q];
    }
    if (n < a.N) {
      if (a.bias) s += __bfloat162float(a.bias[n]);
      static_cast<O*>(a.out)[(size_t)(e >> 7) * a.N + n] = (O)s;
    }
  }
  cluster_sync_all();                                      // nobody leaves while its sums are being read
  if (*(volatile int*)&s_abort) {                          // copies in flight get time to land
    const unsigned long long t0 = gtime_ns();
    while (gtime_ns() - t0 < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) { tc_fence_after(); tmem_dealloc_cta(tmem, COLS); }
}

// ------------------------------------------------------------------ host
typedef void (*FewFn)(FewArgs);
struct FewVariant { int t, quant, f32; FewFn fn; int smem; };
#define V_(T, Q, F, O) {T, Q, F, fp8_few_kernel<T, Q != 0, O>, FewSmem<T>::DYNAMIC}
static const FewVariant g_few[] = {V_(16, 0, 0, bf16), V_(32, 0, 0, bf16), V_(64, 0, 0, bf16), V_(16, 0, 1, float), V_(32, 0, 1, float), V_(64, 0, 1, float),
                                   V_(16, 1, 0, bf16), V_(32, 1, 0, bf16), V_(64, 1, 0, bf16), V_(16, 1, 1, float), V_(32, 1, 1, float), V_(64, 1, 1, float)};
#undef V_

static int few_ready(int dev) {
  static std::mutex mu;
  static bool ready[64] = {false};
  std::lock_guard<std::mutex> l(mu);
  if (ready[dev]) return 0;
  for (const FewVariant& v : g_few) if (cudaFuncSetAttribute((const void*)v.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, v.smem) != cudaSuccess) return -4;
  ready[dev] = true;
  return 0;
}

// x: A in bf16 (rows on 16-byte boundaries, K a multiple of 8), or null: values a with scales sa
int fp8_few(const bf16* x, long long stride, const void* a, const void* sa, const void* b, const void* sb, const void* bias, void* out, int f32, int M, int N, int K, int splits, void* stream) {
  int dev = 0; cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return -6;
  const int rc = few_ready(dev); if (rc) return rc;
  const FewVariant* v = nullptr;
  for (const FewVariant& c : g_few) if (!v && c.t >= M && c.quant == (x != nullptr) && c.f32 == (f32 != 0)) v = &c;
  if (!v) return -1;
  FewArgs g;
  memset(&g, 0, sizeof g);
  g.x = x; g.stride = stride; g.bias = (const bf16*)bias; g.out = out; g.M = M; g.N = N; g.K = K; g.kb = (K + 127) / 128; g.k4 = (g.kb + 3) / 4;
  const int tiles = (N + 127) / 128;
  if (!splits) for (splits = 1; splits < 8 && 2 * splits <= g.kb && tiles * splits * 2 <= 2 * 148; splits *= 2) {}
  if (splits > g.kb) return -1;
  g.splits = splits;
  const uint64_t kp = 128ull * g.kb;
  if (!fp8_map(&g.tw, 1, b, N, kp, 128, 128, true) || !fp8_map(&g.sw, 4, sb, (uint64_t)tiles * g.k4, 128, 1, 128, false)) return -3;
  if (x) { g.tx = g.tw; g.sx = g.sw; }
  else if (!fp8_map(&g.tx, 1, a, M, kp, v->t, 128, true) || !fp8_map(&g.sx, 4, sa, g.k4, 128, 1, 128, false)) return -3;
  g.status = status_word(STATUS_GEMM);
  if (!g.status) return -7;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * splits); cfg.blockDim = dim3(FEW_THREADS); cfg.dynamicSmemBytes = v->smem; cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension; at[1].val.clusterDim.x = splits; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
  cfg.attrs = at; cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, v->fn, g) == cudaSuccess ? 0 : -5;
}

}  // namespace piccl_ops
