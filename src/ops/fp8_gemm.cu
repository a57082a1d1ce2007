// C[M, N] = A[M, K] B[N, K]^T + bias, operands in the 8-bit format of fp8.cuh, on CTA pairs: tcgen05.mma kind::mxf8f6f4, which multiplies by the scales of both
// operands' blocks while it adds to fp32 accumulators in TMEM.
//
// The core is that of sm100_gemm_pair.cuh at a byte an element: a pair has 2 x 128 rows and TN columns, CTA v stages its own rows of A and half of the columns of B, k-blocks of
// 128 (a 128-byte swizzled row each).  A block's scales: 512 bytes of A's 128 rows and of each 128 of B's columns hold four k-blocks; they come by TMA with every fourth k-block,
// tcgen05.cp brings them into 4 columns of TMEM each, and the instruction names the byte of the word that is its block's.
//
// What bounds it: from K of some 2000 on the power that the chip may draw (8192 x 8192 x 3584 168 us when called once, 191 at 1.14 GHz in a loop, 2.5 PFLOP/s).  At K = 1024 a tile of 256 columns takes 5300 clocks, its
// MMAs 4100: the rest is the way from the last MMA to the epilogue's first 32 columns and back (8192 x 4096 x 1024 34 us).  Small ones take some 3 us of ramp, first loads and last epilogue: 1024 x 1024 x 1024 4.8 us,
// 2331 x 768 x 2304 7.2.  Width of tiles by the number of rounds that it takes and the cost of a tile, in piccl_ops_fp8_gemm.
#include <cstring>
#include <mutex>
#include "../include/sm100_gemm_pair.cuh"
#include "fp8.cuh"
#include "fp8_mma.cuh"
#include "piccl_ops.h"

namespace piccl_ops {

using namespace sm100;

struct Fp8Args {
  CUtensorMap ta, tb, sa, sb, tc;
  const bf16* bias;
  void* out;
  int M, N, kb, k4, store_tma, bias_words;       // k-blocks of 128, words of four of them
  int* status;
};

constexpr int FP8_BM = 128, FP8_BK = 128, FP8_THREADS = 320;
constexpr uint32_t kScaleCol = 496;        // TMEM columns: accumulators from 0 on, scales of A 4 from here, of B 8

// AR: rows of A that are staged.  A product of at most 64 rows stages 64: the MMA reads 128 all the same, and what it finds beyond (the next stage) goes into rows that nobody reads.
template <int TN, int STAGES, int AR>
struct Fp8Smem {
  static constexpr int A_BYTES = AR * FP8_BK, B_BYTES = TN / 2 * FP8_BK, STAGE = A_BYTES + B_BYTES;
  static constexpr int NSF = TN > 128 ? 3 : 2, SF_BYTES = 512 * NSF;      // atoms of A's rows and of B's columns
  static constexpr int B_OFF = STAGES * A_BYTES, SF_OFF = STAGES * STAGE, STAGING_OFF = (SF_OFF + STAGES * SF_BYTES + 1023) / 1024 * 1024;
  static constexpr int BAR_OFF = STAGING_OFF + PAIR_EPI_WARPS * PAIR_STAGING;
  static constexpr int TOTAL = BAR_OFF + (2 * STAGES + 4) * 8 + 16, DYNAMIC = TOTAL + 1024;
  static_assert(DYNAMIC <= 232448, "more shared memory than a CTA can have");
  static_assert(STAGES * B_BYTES >= FP8_BM * FP8_BK - A_BYTES, "what is read beyond the last stage of A is there");
};

// 128 bytes of a row of the result
template <typename O> struct OutPiece;
template <> struct OutPiece<bf16> {
  static constexpr int COLS = 64;
  static __device__ __forceinline__ void stage(uint8_t* row, int r, const float (&v)[64]) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      float f[8];
#pragma unroll
      for (int q = 0; q < 8; q++) f[q] = v[8 * j + q];
      *reinterpret_cast<bf16x8*>(row + ((j ^ (r & 7)) << 4)) = pack8(f);
    }
  }
};
template <> struct OutPiece<float> {
  static constexpr int COLS = 32;
  static __device__ __forceinline__ void stage(uint8_t* row, int r, const float (&v)[32]) {
#pragma unroll
    for (int j = 0; j < 8; j++) *reinterpret_cast<float4*>(row + ((j ^ (r & 7)) << 4)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  }
};
// Rows of a result that do not start on 16 bytes, which no TMA store takes: a warp writes a row at a time, a word of 4 bytes a lane, from words of several rows that it has loaded.  Rows of bf16 that begin in the
// middle of a word are moved by half a word, their first and last value written on their own.  What it costs is the instructions and their latencies, not the sectors that are written in part: 2331 x 50257 x 768
// takes 127 us, 85 without this and 102 where 50256 columns go by TMA; with the questions which rows, columns and halves are there asked of each row 150, row by row 208.
__device__ __forceinline__ uint32_t staged_word(const uint8_t* staging, int r, int lane) {
  return *reinterpret_cast<const uint32_t*>(staging + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
}
__device__ __forceinline__ void store_rows(const uint8_t* staging, float* out, size_t stride, int rows, int left, int lane) {
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += 16) {
    uint32_t w[16];
#pragma unroll
    for (int r = 0; r < 16; r++) w[r] = staged_word(staging, r0 + r, lane);
#pragma unroll
    for (int r = 0; r < 16; r++) if (r0 + r < rows && lane < left) out[(r0 + r) * stride + lane] = __uint_as_float(w[r]);
  }
}
// A piece of which all rows and columns are there.  FIRST: its first row begins in the middle of a word, TURNS: every other row does.
__device__ __forceinline__ void store_if(void* p, uint32_t x, bool there) { asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.global.b32 [%0], %1;\n\t}" ::"l"(p), "r"(x), "r"((uint32_t)there) : "memory"); }
__device__ __forceinline__ void store_half_if(void* p, uint32_t x, bool there) {
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.global.b16 [%0], h;\n\t}" ::"l"(p), "r"(x), "r"((uint32_t)there) : "memory");
}
template <bool FIRST, bool TURNS> __device__ __forceinline__ void store_whole_rows(const uint8_t* staging, bf16* out, size_t stride, int lane) {
  const bool inner = lane < 31, end = lane == 0 || lane == 31;
  char* o = reinterpret_cast<char*>(out) + 4 * lane;
  const int to_end = lane == 0 ? 0 : 2;
#pragma unroll 1
  for (int r0 = 0; r0 < 32; r0 += 8) {
    uint32_t w[8], n[8];
#pragma unroll
    for (int r = 0; r < 8; r++) w[r] = staged_word(staging, r0 + r, lane);
#pragma unroll
    for (int r = 0; r < 8; r++) if (FIRST != (TURNS && (r & 1))) n[r] = __shfl_down_sync(0xffffffffu, w[r], 1);
#pragma unroll
    for (int r = 0; r < 8; r++, o += 2 * stride) {
      if (FIRST != (TURNS && (r & 1))) {
        store_if(o + 2, __funnelshift_r(w[r], n[r], 16), inner);
        store_half_if(o + to_end, lane == 0 ? w[r] : w[r] >> 16, end);
      } else *reinterpret_cast<uint32_t*>(o) = w[r];
    }
  }
}
__device__ __forceinline__ bool store_whole(const uint8_t* staging, bf16* out, size_t stride, int rows, int left, int lane) {
  if (rows < 32 || left < 64) return false;
  const bool first = reinterpret_cast<uintptr_t>(out) >> 1 & 1;
  if (stride & 1) { if (first) store_whole_rows<true, true>(staging, out, stride, lane); else store_whole_rows<false, true>(staging, out, stride, lane); }
  else if (first) store_whole_rows<true, false>(staging, out, stride, lane); else store_whole_rows<false, false>(staging, out, stride, lane);
  return true;
}
__device__ __forceinline__ void store_rows(const uint8_t* staging, bf16* out, size_t stride, int rows, int left, int lane) {
  if (store_whole(staging, out, stride, rows, left, lane)) return;
#pragma unroll 1
  for (int r0 = 0; r0 < 32; r0 += 16) {
    uint32_t w[16], n[16];
#pragma unroll
    for (int r = 0; r < 16; r++) w[r] = staged_word(staging, r0 + r, lane);
#pragma unroll
    for (int r = 0; r < 16; r++) n[r] = __shfl_down_sync(0xffffffffu, w[r], 1);
#pragma unroll
    for (int r = 0; r < 16; r++) {
      uint16_t* const o = reinterpret_cast<uint16_t*>(out + (r0 + r) * stride);
      const int odd = (int)(reinterpret_cast<uintptr_t>(o) >> 1) & 1, c = 2 * lane + odd;
      const uint32_t x = odd ? __funnelshift_r(w[r], n[r], 16) : w[r];
      const bool there = r0 + r < rows, whole = c + 1 < left && c < 63;
      if (there && whole) *reinterpret_cast<uint32_t*>(o + c) = x;
      if (there && !whole && c < left) o[c] = (uint16_t)x;
      if (there && odd && lane == 0) o[0] = (uint16_t)w[r];
    }
  }
}

// A tile's sum is one unit, or several that the epilogue adds up: the tensor core cuts its fp32 sums off where an fma would round them, always toward zero, which over K / 32 steps loses
// 2^-25 K / 48 of a sum of random signs (measured 1.6e-6 at K = 2331).  That is nothing to a result in bf16; one in fp32 is added up from units of 1024 k, rounded, in registers.
constexpr int kUnit = 8;           // k-blocks (tiles of 128 columns at most: 64 sums a thread; 128 do not fit beside the rest into the 168 registers that ten warps can have)

// TMEM has 512 columns: two accumulators of 256 and the scales do not fit.  They overlap in 16 columns: the MMAs of the next unit wait until the epilogue has those in registers (its warps
// take the piece with them first), and not for the rest of the tile.
template <int TN, int STAGES, int AR, typename O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(FP8_THREADS, 1) fp8_pair_kernel(const __grid_constant__ Fp8Args a) {
  typedef Fp8Smem<TN, STAGES, AR> L;
  constexpr bool OVERLAP = TN > 240, ADD = sizeof(O) == 4;
  static_assert(!(OVERLAP && ADD) && TN >= 64, "128 sums a thread do not fit; scales lie at even columns");
  constexpr uint32_t ACC = OVERLAP ? 240 : TN;            // columns between the accumulators
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ int s_abort;
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* const full = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t *const empty = full + STAGES, *const tmem_full = empty + STAGES, *const tmem_empty = tmem_full + 2;
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, v = (int)cluster_ctarank();
  const int num_m = (a.M + 255) / 256, num_n = (a.N + TN - 1) / TN, num_tiles = num_m * num_n, first = blockIdx.x >> 1, stride = gridDim.x >> 1;
  const int units = ADD ? (a.kb + kUnit - 1) / kUnit : 1;
  auto tile = [&](int t, int& m_blk, int& n_blk) {         // bands of 16 row tiles, as in gemm_sm100.cu
    const int per_band = 16 * num_n, band = t / per_band, within = t % per_band, rows = min(16, num_m - band * 16);
    m_blk = 2 * (band * 16 + within % rows) + v; n_blk = within / rows;
  };
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int s = 0; s < STAGES; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int i = 0; i < 2; i++) { mbar_init(&tmem_full[i], 1); mbar_init(&tmem_empty[i], 2 * PAIR_EPI_WARPS); }
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc_pair(tmem_slot, 512); tmem_relinquish_pair(); }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_begin();

  if (warp == 0) {
    const bool issuer = elect_one();
    int stage = 0; uint32_t phase = 0;
    for (int t = first; t < num_tiles && !*(volatile int*)&s_abort; t += stride) {
      int m_blk, n_blk; tile(t, m_blk, n_blk);
      bool ok = true;
      for (int kb = 0; kb < a.kb; kb++) {
        if (!mbar_wait(&empty[stage], phase ^ 1, &s_abort, kPairWaitLimitNs)) { if (issuer) atomicExch(a.status, 11); ok = false; break; }
        uint8_t *const pa = smem + stage * L::A_BYTES, *const pb = smem + L::B_OFF + stage * L::B_BYTES, *const ps = smem + L::SF_OFF + stage * L::SF_BYTES;
        if (issuer) {
          const bool scales = (kb & 3) == 0;
          if (v == 0) mbar_arrive_expect_tx(&full[stage], 2 * (L::STAGE + (scales ? L::SF_BYTES : 0)));
          tma_load_2d_pair(pa, &a.ta, kb * FP8_BK, m_blk * FP8_BM, &full[stage]);
          tma_load_2d_pair(pb, &a.tb, kb * FP8_BK, n_blk * TN + v * (TN / 2), &full[stage]);
          if (scales) {
            const int w = kb >> 2;
            tma_load_2d_pair(ps, &a.sa, 0, m_blk * a.k4 + w, &full[stage]);
            tma_load_2d_pair(ps + 512, &a.sb, 0, (n_blk * TN >> 7) * a.k4 + w, &full[stage]);
            if (TN > 128) tma_load_2d_pair(ps + 1024, &a.sb, 0, ((n_blk * TN >> 7) + 1) * a.k4 + w, &full[stage]);
          }
        }
        __syncwarp();
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
      if (!ok) break;
    }
  } else if (warp == 1) {
    if (v == 0) {
      const bool issuer = elect_one();
      constexpr uint32_t idesc = make_idesc_mxf8(256, TN);
      const uint64_t da0 = make_smem_desc_k128(smem), db0 = make_smem_desc_k128(smem + L::B_OFF), ds0 = make_smem_desc_scales(smem + L::SF_OFF);
      const uint32_t sfa = tmem + kScaleCol, sfb = sfa + 4;
      int stage = 0; uint32_t phase = 0; int local = 0;
      bool ok = true;
      for (int t = first; ok && t < num_tiles && !*(volatile int*)&s_abort; t += stride) {
        int m_blk, n_blk; tile(t, m_blk, n_blk);
        const uint32_t sfb_t = sfb + (TN == 64 ? 2 * (n_blk & 1) : 0);      // where in its 128 columns the tile begins (an even column of TMEM: tiles of 32 cannot be)
        for (int u = 0; ok && u < units; u++, local++) {
          const int acc = local & 1;
          // overlapping: the edge of the unit before is in registers, and with it all of the one before that; else: this accumulator's unit is
          if (OVERLAP ? local > 0 && !mbar_wait(&tmem_empty[0], (local - 1) & 1, &s_abort, kPairWaitLimitNs) : !mbar_wait(&tmem_empty[acc], ((local >> 1) & 1) ^ 1, &s_abort, kPairWaitLimitNs)) {
            if (issuer) atomicExch(a.status, 12);
            ok = false; break;
          }
          tc_fence_after();
          const uint32_t d = tmem + acc * ACC;
          const int kb0 = ADD ? u * kUnit : 0, kb1 = ADD ? min(a.kb, kb0 + kUnit) : a.kb;
          for (int kb = kb0; kb < kb1; kb++) {
            if (!mbar_wait(&full[stage], phase, &s_abort, kPairWaitLimitNs)) { if (issuer) atomicExch(a.status, 13); ok = false; break; }
            tc_fence_after();
            const uint64_t da = desc_advance(da0, stage * L::A_BYTES), db = desc_advance(db0, stage * L::B_BYTES);
            if (issuer) {
              if ((kb & 3) == 0) {
                const uint64_t ds = desc_advance(ds0, stage * L::SF_BYTES);
                scales_to_tmem_pair(sfa, ds);
                scales_to_tmem_pair(sfb, desc_advance(ds, 512));
                if (TN > 128) scales_to_tmem_pair(sfb + 4, desc_advance(ds, 1024));
              }
#pragma unroll
              for (int k = 0; k < FP8_BK / 32; k++) umma_mxf8_pair(d, desc_advance(da, k * 32), desc_advance(db, k * 32), idesc | idesc_bytes(kb & 3, kb & 3), sfa, sfb_t, kb != kb0 || k != 0);
              umma_commit_pair(&empty[stage]);
            }
            __syncwarp();
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
          }
          if (ok && issuer) umma_commit_pair(&tmem_full[acc]);
          __syncwarp();
        }
      }
    }
  } else {
    typedef OutPiece<O> P;
    constexpr int PIECES = TN / P::COLS, PER = PIECES >= 2 ? PIECES / 2 : 1;
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    uint8_t* const staging = smem + L::STAGING_OFF + (warp - 2) * PAIR_STAGING;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    int local = 0;
    bool ok = true;
    for (int t = first; ok && t < num_tiles; t += stride) {
      int m_blk, n_blk; tile(t, m_blk, n_blk);
      const int row0 = m_blk * FP8_BM + quarter * 32;
      const bool mine = row0 < a.M && (PIECES >= 2 || half == 0);
      // a piece of the thread's row on its way out
      auto ship = [&](float (&x)[P::COLS], int pc) {
        const int col = n_blk * TN + pc * P::COLS;
        if (col >= a.N) return;
        if (a.bias) {
          if (col + P::COLS <= a.N && a.bias_words) {
#pragma unroll
            for (int j = 0; j < P::COLS; j += 8) {
              float f[8]; unpack8(*reinterpret_cast<const bf16x8*>(a.bias + col + j), f);
#pragma unroll
              for (int q = 0; q < 8; q++) x[j + q] += f[q];
            }
          } else {
#pragma unroll
            for (int j = 0; j < P::COLS; j++) x[j] += __bfloat162float(a.bias[min(col + j, a.N - 1)]);
          }
        }
        if (lane == 0) bulk_wait_read_all();               // the last store has been read out of the staging buffer
        __syncwarp();
        P::stage(staging + lane * 128, lane, x);
        if (a.store_tma) {
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) { tma_store_2d(&a.tc, staging, col, row0); bulk_commit(); }
          __syncwarp();
        } else {
          __syncwarp();
          store_rows(staging, static_cast<O*>(a.out) + (size_t)row0 * a.N + col, a.N, a.M - row0, a.N - col, lane);
          __syncwarp();
        }
      };
      // waits for a unit; true: this warp's columns are among those that the accumulators share, and it reports when it has them
      auto arrived = [&](bool& edge) {
        edge = OVERLAP && half == ((local & 1) ^ 1) && mine;
        if (!mbar_wait(&tmem_full[local & 1], (local >> 1) & 1, &s_abort, kPairWaitLimitNs)) { atomicExch(a.status, 14); return false; }
        tc_fence_after();
        if (OVERLAP && !edge && lane == 0) mbar_arrive_leader(&tmem_empty[0]);
        __syncwarp();                                      // tcgen05.ld, which comes next, wants the whole warp at one place: so after everything that one lane does
        return true;
      };
      auto taken = [&](uint64_t* bar) { tc_fence_before(); __syncwarp(); if (lane == 0) mbar_arrive_leader(bar); __syncwarp(); };
      bool edge;
      if constexpr (ADD) {
        float x[PER][P::COLS];
#pragma unroll
        for (int i = 0; i < PER; i++)
#pragma unroll
          for (int j = 0; j < P::COLS; j++) x[i][j] = 0.f;
#pragma unroll 1
        for (int u = 0; u < units; u++, local++) {
          if (!arrived(edge)) { ok = false; break; }
          if (mine) {
#pragma unroll
            for (int i = 0; i < PER; i++)
#pragma unroll
              for (int q = 0; q < P::COLS / 16; q++) {     // few columns at a time: the sums leave few registers
                uint32_t r[16];
                tmem_ld_32x16(lanes + (local & 1) * ACC + (half ? PIECES - 1 - i : i) * P::COLS + 16 * q, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; j++) x[i][16 * q + j] += __uint_as_float(r[j]);
              }
          }
          taken(&tmem_empty[local & 1]);
        }
        if (ok && mine) {
#pragma unroll
          for (int i = 0; i < PER; i++) ship(x[i], half ? PIECES - 1 - i : i);
        }
      } else {
        if (!arrived(edge)) { ok = false; break; }
        if (mine) {
#pragma unroll 1
          for (int i = 0; i < PER; i++) {
            const int pc = half ? PIECES - 1 - i : i;
            float x[P::COLS];
            auto load = [&](int q) { tmem_ld_32x32(lanes + (local & 1) * ACC + pc * P::COLS + 32 * q, reinterpret_cast<uint32_t (&)[32]>(x[32 * q])); };
            // the columns that the accumulators share first: the last ones of the upper half, the first ones of the lower
            if (half) load(1); else load(0);
            if (i == 0 && edge) { tmem_ld_wait(); taken(&tmem_empty[0]); }
            if (half) load(0); else load(1);
            tmem_ld_wait();
            ship(x, pc);
          }
        }
        if (!OVERLAP) taken(&tmem_empty[local & 1]);
        local++;
      }
    }
  }
  // the ending of gemm_pair_persistent: nobody leaves while the other CTA may still touch its shared memory or barriers
  tc_fence_before();
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  if (warp >= 2 && lane == 0) bulk_wait_read_all();
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (*(volatile int*)&s_abort) {
    const unsigned long long t0 = gtime_ns();
    while (gtime_ns() - t0 < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  __syncwarp();
  if (warp == 1) { tc_fence_after(); tmem_dealloc_pair(tmem, 512); }
}

// ------------------------------------------------------------------ host
typedef void (*Fp8Fn)(Fp8Args);
struct Fp8Variant { int tn, ar, f32; Fp8Fn fn; int smem; };
#define V_(TN, ST, AR, F, O) {TN, AR, F, fp8_pair_kernel<TN, ST, AR, O>, Fp8Smem<TN, ST, AR>::DYNAMIC}
static const Fp8Variant g_fp8[] = {V_(256, 5, 128, 0, bf16), V_(128, 7, 128, 0, bf16), V_(64, 8, 128, 0, bf16), V_(64, 14, 64, 0, bf16),
                                   V_(128, 7, 128, 1, float), V_(64, 8, 128, 1, float), V_(64, 14, 64, 1, float)};
#undef V_
static int g_fp8_pairs[64] = {0};

static int fp8_ready(int dev) {
  static std::mutex mu;
  std::lock_guard<std::mutex> l(mu);
  if (g_fp8_pairs[dev]) return 0;
  for (const Fp8Variant& v : g_fp8) if (cudaFuncSetAttribute((const void*)v.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, v.smem) != cudaSuccess) return -4;
  int sms = 148; cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sms / 2 * 2); cfg.blockDim = dim3(FP8_THREADS); cfg.dynamicSmemBytes = g_fp8[0].smem;
  cudaLaunchAttribute at; memset(&at, 0, sizeof at);
  at.id = cudaLaunchAttributeClusterDimension; at.val.clusterDim.x = 2; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
  cfg.attrs = &at; cfg.numAttrs = 1;
  int active = 0, n = sms / 2;
  if (cudaOccupancyMaxActiveClusters(&active, g_fp8[0].fn, &cfg) == cudaSuccess && active > 0) n = active < n ? active : n;
  else cudaGetLastError();
  g_fp8_pairs[dev] = n;
  return 0;
}

}  // namespace piccl_ops

using namespace piccl_ops;

static bool few_takes(const void* x, int fp32, long long stride, int M, int N, long long K) {
  return fp8_few_takes(M, N, K, false) && !fp32 && K % 8 == 0 && stride % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
}

extern "C" {

// a [M, K], b [N, K], K a multiple of 128, with their scales; out [M, N] bf16 or fp32, rows next to each other; bias [N] bf16 or null.  force_tn: 0, or the tile's width (for tests).
int piccl_ops_fp8_gemm(const void* a, const void* sa, const void* b, const void* sb, const void* bias, void* out, int f32, int M, int N, long long K, int force_tn, void* stream) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 128 || K > 0x7fffff00ll || M > 0x7fffff00 || N > 0x7fffff00) return -1;
  for (const void* p : {a, sa, b, sb}) if (!p || (reinterpret_cast<uintptr_t>(p) & 15)) return -2;
  if (!out || (reinterpret_cast<uintptr_t>(out) & (f32 ? 3 : 1)) || (reinterpret_cast<uintptr_t>(bias) & 1)) return -2;
  if (!force_tn && fp8_few_takes(M, N, K, true)) return fp8_few(nullptr, 0, a, sa, b, sb, bias, out, f32, M, N, (int)K, stream);
  int dev = 0; cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return -6;
  const int rc = fp8_ready(dev); if (rc) return rc;
  const long row_tiles = (M + 255) / 256;
  const Fp8Variant* v = nullptr; double best = 0;
  for (const Fp8Variant& c : g_fp8) {
    if (c.f32 != (f32 != 0) || (force_tn && c.tn != force_tn) || (c.ar == 64) != (M <= 64 && c.tn <= 64)) continue;
    const long tiles = row_tiles * ((N + c.tn - 1) / c.tn);
    const double cost = (double)((tiles + g_fp8_pairs[dev] - 1) / g_fp8_pairs[dev]) * (c.tn == 256 ? 136 : c.tn == 128 ? 84 : 70);
    if (!v || cost < best) { v = &c; best = cost; }
  }
  if (!v || (double)row_tiles * ((N + v->tn - 1) / v->tn) > 0x7fffffff) return -1;
  Fp8Args g;
  memset(&g, 0, sizeof g);
  g.M = M; g.N = N; g.kb = (int)(K / 128); g.k4 = (g.kb + 3) / 4; g.bias = (const bf16*)bias; g.out = out;
  const int esz = f32 ? 4 : 2;
  g.store_tma = (size_t)N * esz % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  if (!fp8_map(&g.ta, 1, a, M, K, v->ar, FP8_BK, true) || !fp8_map(&g.tb, 1, b, N, K, v->tn / 2, FP8_BK, true) ||
      !fp8_map(&g.sa, 4, sa, (uint64_t)((M + 127) / 128) * g.k4, 128, 1, 128, false) || !fp8_map(&g.sb, 4, sb, (uint64_t)((N + 127) / 128) * g.k4, 128, 1, 128, false)) return -3;
  if (g.store_tma && !fp8_map(&g.tc, esz, out, M, N, 32, 128 / esz, true)) return -3;
  g.bias_words = reinterpret_cast<uintptr_t>(bias) % 16 == 0;
  g.status = status_word(STATUS_GEMM);
  if (!g.status) return -7;
  const long tiles = row_tiles * ((N + v->tn - 1) / v->tn);
  const int pairs = (int)(tiles < g_fp8_pairs[dev] ? tiles : g_fp8_pairs[dev]);
  return launch_pdl(v->fn, dim3(2 * pairs), dim3(FP8_THREADS), v->smem, (cudaStream_t)stream, g) == cudaSuccess ? 0 : -5;
}


// out [M, N] = x [M, K] w [N, K]^T + bias, x bf16 (or fp32) with rows `stride` elements apart; keep, keep_s: null, or room for x along its columns in 8 bits ([K, M up to 128]).
// scratch, scratch_s: room for x in 8 bits, or null where piccl_ops_fp8_linear_scratch says 0.  Returns the number of launches, or a negative code.
int piccl_ops_fp8_linear_scratch(const void* x, int fp32, long long stride, int M, int N, long long K, int keep) { return keep || !few_takes(x, fp32, stride, M, N, K); }
int piccl_ops_fp8_linear(const void* x, int fp32, long long stride, const void* w, const void* sw, const void* bias, void* out, int f32, void* scratch, void* scratch_s, void* keep, void* keep_s, int M,
                         int N, long long K, void* stream) {
  if (M <= 0 || N <= 0 || K <= 0 || K > 0x7fffff00ll || stride < K) return -1;
  if (!piccl_ops_fp8_linear_scratch(x, fp32, stride, M, N, K, keep != nullptr)) {
    for (const void* p : {x, w, sw}) if (!p || (reinterpret_cast<uintptr_t>(p) & 15)) return -2;
    if (!out || (reinterpret_cast<uintptr_t>(out) & (f32 ? 3 : 1)) || (reinterpret_cast<uintptr_t>(bias) & 1)) return -2;
    const int rc = fp8_few((const bf16*)x, stride, nullptr, nullptr, w, sw, bias, out, f32, M, N, (int)K, stream);
    return rc ? rc : 1;
  }
  if (!scratch || !scratch_s) return -2;
  int rc = piccl_ops_fp8_quantize(x, fp32, M, K, stride, scratch, scratch_s, keep, keep_s, 0, stream);
  if (!rc) rc = piccl_ops_fp8_gemm(scratch, scratch_s, w, sw, bias, out, f32, M, N, (K + 127) / 128 * 128, 0, stream);
  return rc > 0 ? -rc - 100 : rc ? rc : 2;
}

}  // extern "C"
