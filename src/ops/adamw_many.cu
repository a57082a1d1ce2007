// AdamW over many tensors in one launch, moments in fp32 or in 8 bits.
//
//   g' = g * gscale     m' = b1 m + (1 - b1) g'     v' = b2 v + (1 - b2) g' g'     w' = w (1 - lr wd) - lr (m' / (1 - b1^t)) / (sqrt(v' / (1 - b2^t)) + eps)
//
// In 8 bits the moments lie as e4m3 with a power of two for each block of 128 elements (fp8.cuh), the second one as its root: a root has half the range (e4m3's smallest step is
// 2^-18 of a block's largest value, 2^-36 of the largest v) and is what the update divides by.  Both are rounded stochastically, up with the probability of the part cut off.
// Rounded to nearest they would stand still: with b2 = 0.999 a root changes by 0.05 % a step, and e4m3's half step is 3 to 6 %.  A root that is not zero does not become zero, or the
// update of an element whose gradients are 2^-18 of its block's largest would divide by eps alone.  The random bits are a hash of the element's place, the step and a seed, so a run can be
// repeated bit by bit; for the same reason the state's arithmetic is in single roundings (no fma).
#include "fp8.cuh"

namespace piccl_ops {

// A tensor: addresses, elements, its first block of 128 in the state, what it is.  Mirrored in piccl_b200/ops/optimizer.py.
struct AdamTensor {
  void* p; float* master; const void* g;
  long long n, block;
  int flags, pad;
};
enum { ADAM_DECAY = 1, ADAM_P_F32 = 2, ADAM_G_F32 = 4, ADAM_WORDS = 8 };      // WORDS: every address on a boundary of four elements

struct AdamArgs {
  const AdamTensor* tensors; int count; long long blocks;
  void *m, *v; uint8_t *ms, *vs;
  float lr, b1, c1, b2, c2, eps, wd; double lb1, lb2;      // c: 1 - b; lb: logarithms
  float gscale; const float* gscale_dev;
  int* step; unsigned* ticket; uint32_t seed;
};

__device__ __forceinline__ uint32_t random_bits(uint32_t place, uint32_t key) {
  uint32_t h = place * 0x9E3779B9u + key;      // the golden ratio, then the roots of 3 and 2: odd numbers without a pattern
  h = (h ^ (h >> 16)) * 0xBB67AE85u;
  h = (h ^ (h >> 15)) * 0x6A09E667u;
  return h ^ (h >> 16);
}
__device__ __forceinline__ void e4m3_values(uint32_t four, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(four >> (16 * i)), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    v[2 * i] = f.x; v[2 * i + 1] = f.y;
  }
}
// x / scale rounded to e4m3, up with probability (part cut off) * 2^16 of bits 0..15 of `bits`
template <bool POSITIVE> __device__ __forceinline__ float stochastic(float x, float f, uint32_t bits) {
  const float t = x * f, a = fabsf(t), low = a < 0.015625f ? 0.015625f : 0.f;      // below 2^-6 the steps are those of [2^-6, 2^-5)
  float z = __uint_as_float((__float_as_uint(a + low) + (bits << 4)) & 0xfff00000u) - low;
  if (POSITIVE && a > 0.f) z = fmaxf(z, 0.001953125f);
  return finite_bits(x) | (x == 0.f) ? copysignf(z, t) : __uint_as_float(0x7fffffffu);
}
template <bool POSITIVE> __device__ __forceinline__ uint32_t round_block(const float (&x)[4], const uint32_t (&bits)[4], uint32_t& byte) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 4; e++) top = max(top, finite_bits(x[e]));
  byte = scale_byte(__reduce_max_sync(0xffffffffu, top));
  const float f = scale_inverse(byte);
  float z[4];
#pragma unroll
  for (int e = 0; e < 4; e++) z[e] = stochastic<POSITIVE>(x[e], f, POSITIVE ? bits[e] >> 16 : bits[e] & 0xffffu);
  return e4m3_pair(z[0], z[1]) | e4m3_pair(z[2], z[3]) << 16;
}

// A warp has a block of 128 elements, a lane four of them.
template <bool BITS8>
__global__ void __launch_bounds__(256) adamw_many_kernel(const AdamArgs a) {
  pdl_begin();
  __shared__ float s_c[2];
  const int t = *(volatile int*)a.step + 1;
  if (threadIdx.x == 0) {
    s_c[0] = (float)(1.0 / -expm1(t * a.lb1));
    s_c[1] = (float)(1.0 / sqrt(-expm1(t * a.lb2)));
  }
  __syncthreads();
  const float rc1 = s_c[0], rc2 = s_c[1], gscale = a.gscale_dev ? a.gscale * *a.gscale_dev : a.gscale;
  const uint32_t key = a.seed + (uint32_t)t * 0x9E3779B9u;
  const int lane = threadIdx.x & 31;
  const long long stride = gridDim.x * 8ll;
  int at = 0;
  for (long long block = blockIdx.x * 8ll + (threadIdx.x >> 5); block < a.blocks; block += stride) {
    if (at + 1 < a.count && a.tensors[at + 1].block <= block) {      // the last tensor that begins at or before the block
      int lo = at + 1, hi = a.count;
      while (hi - lo > 1) { const int mid = (lo + hi) / 2; (a.tensors[mid].block <= block ? lo : hi) = mid; }
      at = lo;
    }
    const AdamTensor& q = a.tensors[at];
    const int flags = q.flags;
    const long long i = (block - q.block) * 128 + lane * 4, s = block * 128 + lane * 4;
    const int left = (int)min(4ll, q.n - i);                          // elements of this lane, none or fewer if not positive
    const bool words = (flags & ADAM_WORDS) && left == 4;
    float g[4] = {0.f, 0.f, 0.f, 0.f}, w[4] = {0.f, 0.f, 0.f, 0.f}, m[4], v[4];
    float* const master = flags & ADAM_P_F32 ? static_cast<float*>(q.p) : q.master;
    if (words) {
      if (flags & ADAM_G_F32) *reinterpret_cast<float4*>(g) = reinterpret_cast<const float4*>(static_cast<const float*>(q.g) + i)[0];
      else {
        const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const bf16*>(q.g) + i);
        g[0] = __uint_as_float(u.x << 16); g[1] = __uint_as_float(u.x & 0xffff0000u); g[2] = __uint_as_float(u.y << 16); g[3] = __uint_as_float(u.y & 0xffff0000u);
      }
      *reinterpret_cast<float4*>(w) = *reinterpret_cast<const float4*>(master + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) if (e < left) {
        g[e] = flags & ADAM_G_F32 ? static_cast<const float*>(q.g)[i + e] : __bfloat162float(static_cast<const bf16*>(q.g)[i + e]);
        w[e] = master[i + e];
      }
    }
    if (BITS8) {
      e4m3_values(static_cast<const uint32_t*>(a.m)[s / 4], m);
      e4m3_values(static_cast<const uint32_t*>(a.v)[s / 4], v);
      const float fm = scale_value(a.ms[block]), fv = scale_value(a.vs[block]);
#pragma unroll
      for (int e = 0; e < 4; e++) { m[e] *= fm; v[e] *= fv; v[e] = __fmul_rn(v[e], v[e]); }
    } else {
      *reinterpret_cast<float4*>(m) = *reinterpret_cast<const float4*>(static_cast<const float*>(a.m) + s);
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(static_cast<const float*>(a.v) + s);
    }
    const float keep = 1.f - a.lr * (flags & ADAM_DECAY ? a.wd : 0.f);
    float r[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float x = __fmul_rn(g[e], gscale);
      m[e] = __fadd_rn(__fmul_rn(a.b1, m[e]), __fmul_rn(a.c1, x));
      v[e] = __fadd_rn(__fmul_rn(a.b2, v[e]), __fmul_rn(__fmul_rn(a.c2, x), x));
      r[e] = __fsqrt_rn(v[e]);
      w[e] = w[e] * keep - a.lr * (m[e] * rc1) / (r[e] * rc2 + a.eps);
    }
    if (words) {
      *reinterpret_cast<float4*>(master + i) = *reinterpret_cast<const float4*>(w);
      if (!(flags & ADAM_P_F32)) {
        __nv_bfloat162 o[2] = {__floats2bfloat162_rn(w[0], w[1]), __floats2bfloat162_rn(w[2], w[3])};
        *reinterpret_cast<uint2*>(static_cast<bf16*>(q.p) + i) = *reinterpret_cast<const uint2*>(o);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) if (e < left) {
        master[i + e] = w[e];
        if (!(flags & ADAM_P_F32)) static_cast<bf16*>(q.p)[i + e] = __float2bfloat16_rn(w[e]);
      }
    }
    if (BITS8) {
      uint32_t bits[4], bm, bv;
#pragma unroll
      for (int e = 0; e < 4; e++) bits[e] = random_bits((uint32_t)s + e, key);
#pragma unroll
      for (int e = 0; e < 4; e++) if (e >= left) { m[e] = 0.f; r[e] = 0.f; }
      const uint32_t om = round_block<false>(m, bits, bm), ov = round_block<true>(r, bits, bv);
      static_cast<uint32_t*>(a.m)[s / 4] = om;
      static_cast<uint32_t*>(a.v)[s / 4] = ov;
      if (lane == 0) { a.ms[block] = bm; a.vs[block] = bv; }
    } else {
      *reinterpret_cast<float4*>(static_cast<float*>(a.m) + s) = *reinterpret_cast<const float4*>(m);
      *reinterpret_cast<float4*>(static_cast<float*>(a.v) + s) = *reinterpret_cast<const float4*>(v);
    }
  }
  __syncthreads();                                        // every thread has read *step
  if (threadIdx.x == 0 && atomicAdd(a.ticket, 1u) == gridDim.x - 1) { *a.ticket = 0; atomicAdd(a.step, 1); }
}

}  // namespace piccl_ops

using namespace piccl_ops;

extern "C" {

// tensors: device array of `count` records in the order of their blocks, which follow each other and cover [0, blocks); m, v: blocks * 128 elements (fp32, or bytes with a byte of scale for each
// block); step: device int, steps done so far, advanced by the launch; ticket: device int that holds zero.  gscale_dev: null, or a device float that multiplies gscale.
int piccl_ops_adamw_many(const void* tensors, int count, long long blocks, int bits8, void* m, void* v, void* ms, void* vs, float lr, double b1, double b2, float eps, float wd, float gscale,
                         const float* gscale_dev, int* step, unsigned* ticket, unsigned seed, void* stream) {
  if (count < 0 || blocks < 0 || !(b1 >= 0 && b1 < 1) || !(b2 >= 0 && b2 < 1)) return -1;
  if ((blocks && (!tensors || !m || !v || (bits8 && (!ms || !vs)))) || !step || !ticket) return -2;
  if ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 15) return -2;
  AdamArgs a{static_cast<const AdamTensor*>(tensors), count, blocks, m, v, (uint8_t*)ms, (uint8_t*)vs, lr, (float)b1, (float)(1 - b1), (float)b2, (float)(1 - b2), eps, wd, log(b1), log(b2),
             gscale, gscale_dev, step, ticket, seed};
  const long long want = (blocks + 7) / 8, most = 148 * 8;
  const unsigned grid = (unsigned)(want < 1 ? 1 : want < most ? want : most);
  const cudaError_t e = launch_pdl(bits8 ? adamw_many_kernel<true> : adamw_many_kernel<false>, dim3(grid), 256, 0, (cudaStream_t)stream, a);
  return e == cudaSuccess ? 0 : (int)e;
}

}  // extern "C"
