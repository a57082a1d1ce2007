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
enum { ADAM_DECAY = 1, ADAM_P_F32 = 2, ADAM_G_F32 = 4, ADAM_WORDS = 8 };      // WORDS: every address on a boundary of 16 bytes

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
__device__ __forceinline__ void e4m3_values(uint32_t four, float f, f32x2 (&v)[2]) {      // times f
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(four >> (16 * i)), __NV_E4M3);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
    v[i] = mul2(pack2(x.x, x.y), both2(f));
  }
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) { float r; asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
__device__ __forceinline__ float min3(float a, float b, float c) { float r; asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
// Where an element's 16 random bits stand among the 20 that are cut off
template <bool ROOT> __device__ __forceinline__ uint32_t random_part(uint32_t r) { return (ROOT ? r >> 16 : r & 0xffffu) << 4; }
// x / scale, at most 448 in magnitude, rounded: what is cut off of its fraction, and the random bits, carry.  Its magnitude is 2^-6 or more: the steps of e4m3 are those of three bits of fraction.
template <bool ROOT> __device__ __forceinline__ float stochastic(float t, uint32_t r) { return __uint_as_float((__float_as_uint(t) + random_part<ROOT>(r)) & 0xfff00000u); }
// The same for any magnitude, and NaN for x that is not finite; a root that is not zero stays so
template <bool ROOT> __device__ __forceinline__ float stochastic_any(float x, float t, uint32_t r) {
  if ((__float_as_uint(x) & 0x7fffffffu) >= kInf) return __uint_as_float(0x7fffffffu);
  const float a = fabsf(t), low = a < 0.015625f ? 0.015625f : 0.f;      // below 2^-6 the steps are those of [2^-6, 2^-5)
  float z = stochastic<ROOT>(a + low, r) - low;
  if (ROOT && a > 0.f) z = fmaxf(z, 0.001953125f);
  return copysignf(z, t);
}
// The byte of a block whose largest value is the root of v: the smallest s for which v <= (448 * 2^s)^2 = 1.53125 * 2^(17 + 2 s).  (A root rounded to fp32 is above 448 * 2^s exactly
// where v is above that, so this is the byte of correctly rounded roots.)
__device__ __forceinline__ uint32_t scale_byte_of_root(uint32_t v_bits) {
  const int e = (int)((v_bits + (0x7fffffu - 0x440000u)) >> 23) - 127 - 17, s = 127 + ((e + 1) >> 1);
  return v_bits < 0x00800000u ? 1u : (uint32_t)s;
}
// Eight of a block's values, by 16 lanes -> their bytes and the block's; of: what the values are the roots of (the values themselves, if they are not roots)
template <bool ROOT> __device__ __forceinline__ uint2 round_block(const f32x2 (&x2)[4], const f32x2 (&of)[4], const uint32_t (&random)[8], uint32_t mask, uint32_t& byte) {
  float x[8], y[8];
#pragma unroll
  for (int i = 0; i < 4; i++) { unpack2(x2[i], x[2 * i], x[2 * i + 1]); unpack2(of[i], y[2 * i], y[2 * i + 1]); }
  float most = max3_nan(fabsf(y[0]), fabsf(y[1]), fabsf(y[2])), least = min3(fabsf(x[0]), fabsf(x[1]), fabsf(x[2]));
#pragma unroll
  for (int e = 3; e < 7; e += 2) { most = max3_nan(most, fabsf(y[e]), fabsf(y[e + 1])); least = min3(least, fabsf(x[e]), fabsf(x[e + 1])); }
  most = max3_nan(most, fabsf(y[7]), fabsf(y[7])); least = fminf(least, fabsf(x[7]));
  uint32_t top = __float_as_uint(most);
  bool odd = __any_sync(mask, top >= kInf);
  if (odd) {
    top = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) top = max(top, finite_bits(y[e]));
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(mask, top, o));
  byte = ROOT ? scale_byte_of_root(top) : scale_byte(top);
  const float f = scale_inverse(byte);
  odd = odd || __any_sync(mask, least * f < 0.015625f);
  float t[8];
#pragma unroll
  for (int i = 0; i < 4; i++) unpack2(mul2(x2[i], both2(f)), t[2 * i], t[2 * i + 1]);
  if (odd) {
#pragma unroll
    for (int e = 0; e < 8; e++) t[e] = stochastic_any<ROOT>(x[e], t[e], random[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) t[e] = stochastic<ROOT>(t[e], random[e]);
  }
  return make_uint2(e4m3_pair(t[0], t[1]) | e4m3_pair(t[2], t[3]) << 16, e4m3_pair(t[4], t[5]) | e4m3_pair(t[6], t[7]) << 16);
}

// Eight elements of a lane as they come from memory
template <bool BITS8> struct AdamRaw {
  static constexpr int S = BITS8 ? 2 : 8;                  // words of a moment
  uint32_t g[8], w[8], m[S], v[S];
  uint32_t fm, fv;                                         // bytes of the moments' scales
};
// The tensor that a lane works on
struct AdamNow {
  void* p; float* master; const void* g;
  long long n, first, end;                                 // elements; its first block, that of the next tensor
  int at, flags;
};
// Where eight elements of it lie
struct AdamPlace {
  float* master; bf16* p;                                  // p: null if the parameters are the masters
  int left, flags;                                         // elements of the lane, at most 8 (not positive: none)
  __device__ __forceinline__ bool words() const { return (flags & ADAM_WORDS) && left == 8; }
};
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[8]) {
  const uint4 a = static_cast<const uint4*>(p)[0], b = static_cast<const uint4*>(p)[1];
  w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
}
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[2]) { const uint2 a = *static_cast<const uint2*>(p); w[0] = a.x; w[1] = a.y; }
__device__ __forceinline__ void store_words(void* p, const uint32_t (&w)[8]) {
  static_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]); static_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

__device__ __forceinline__ void adam_find(const AdamArgs& a, long long block, AdamNow& c) {      // the last tensor that begins at or before the block, from c.at on
  int lo = c.at, hi = a.count;
  while (hi - lo > 1) { const int mid = (lo + hi) / 2; (a.tensors[mid].block <= block ? lo : hi) = mid; }
  const AdamTensor& q = a.tensors[lo];
  c.at = lo; c.flags = q.flags; c.p = q.flags & ADAM_P_F32 ? nullptr : q.p; c.master = q.flags & ADAM_P_F32 ? static_cast<float*>(q.p) : q.master; c.g = q.g; c.n = q.n; c.first = q.block;
  c.end = lo + 1 < a.count ? a.tensors[lo + 1].block : a.blocks;
}
template <bool BITS8> __device__ __forceinline__ AdamPlace adam_load(const AdamArgs& a, AdamNow& c, long long block, int l16, AdamRaw<BITS8>& r) {
  if (block >= c.end) adam_find(a, block, c);
  const long long i = (block - c.first) * 128 + l16 * 8;
  AdamPlace o{c.master + i, c.p ? static_cast<bf16*>(c.p) + i : nullptr, (int)min(8ll, c.n - i), c.flags};
  if (o.words()) {
    if (o.flags & ADAM_G_F32) load_words(static_cast<const float*>(c.g) + i, r.g);
    else { const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(c.g) + i); r.g[0] = u.x; r.g[1] = u.y; r.g[2] = u.z; r.g[3] = u.w; }
    load_words(o.master, r.w);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) { r.g[e] = 0; r.w[e] = 0; }
#pragma unroll
    for (int e = 0; e < 8; e++) if (e < o.left) {
      if (o.flags & ADAM_G_F32) r.g[e] = static_cast<const uint32_t*>(c.g)[i + e];
      else r.g[e >> 1] |= (uint32_t)static_cast<const uint16_t*>(c.g)[i + e] << (16 * (e & 1));
      r.w[e] = __float_as_uint(o.master[e]);
    }
  }
  const long long s = block * 128 + l16 * 8;
  if (BITS8) {
    load_words(static_cast<const uint8_t*>(a.m) + s, r.m);
    load_words(static_cast<const uint8_t*>(a.v) + s, r.v);
    r.fm = a.ms[block]; r.fv = a.vs[block];
  } else {
    load_words(static_cast<const float*>(a.m) + s, r.m);
    load_words(static_cast<const float*>(a.v) + s, r.v);
  }
  return o;
}
// The root of v: in 8 bits the approximate one (2^-23; what it is rounded to has 2^-4), in which v below 2^-126 counts as zero
template <bool BITS8> __device__ __forceinline__ float adam_root(float v) {
  float r;
  if (BITS8) asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); else r = __fsqrt_rn(v);
  return r;
}

// Sixteen lanes have a block of 128 elements, a lane eight of them; the next block's are on their way while one is worked on.
template <bool BITS8>
__global__ void __launch_bounds__(256, BITS8 ? 3 : 2) adamw_many_kernel(const AdamArgs a) {
  pdl_begin();
  __shared__ float s_c[2];
  const int t = *(volatile int*)a.step + 1;
  if (threadIdx.x == 0) {
    s_c[0] = (float)(1.0 / -expm1(t * a.lb1));
    s_c[1] = (float)(1.0 / sqrt(-expm1(t * a.lb2)));
  }
  __syncthreads();
  const float rc2 = s_c[1], gscale = a.gscale_dev ? a.gscale * *a.gscale_dev : a.gscale, lr1 = a.lr * s_c[0];
  const uint32_t key = a.seed + (uint32_t)t * 0x9E3779B9u, mask = 0xffffu << (threadIdx.x & 16);
  const int l16 = threadIdx.x & 15;
  const long long stride = gridDim.x * 16ll;
  long long block = blockIdx.x * 16ll + (threadIdx.x >> 4);
  AdamNow now;
  now.at = 0; now.end = -1;
  AdamRaw<BITS8> r, next;
  AdamPlace o, then;
  if (block < a.blocks) o = adam_load(a, now, block, l16, r);
  for (; block < a.blocks; block += stride, o = then, r = next) {
    if (block + stride < a.blocks) then = adam_load(a, now, block + stride, l16, next);
    f32x2 g[4], m[4], v[4], root[4];
    float w[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      g[i] = o.flags & ADAM_G_F32 ? pack2(__uint_as_float(r.g[2 * i]), __uint_as_float(r.g[2 * i + 1])) : pack2(__uint_as_float(r.g[i] << 16), __uint_as_float(r.g[i] & 0xffff0000u));
      g[i] = mul2(g[i], both2(gscale));
    }
    if (BITS8) {
      const float fm = scale_value(r.fm), fv = scale_value(r.fv);
#pragma unroll
      for (int i = 0; i < 2; i++) {
        e4m3_values(r.m[i], fm, reinterpret_cast<f32x2 (&)[2]>(m[2 * i]));
        e4m3_values(r.v[i], fv, reinterpret_cast<f32x2 (&)[2]>(v[2 * i]));
      }
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = mul2(v[i], v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        m[i] = pack2(__uint_as_float(r.m[2 * i]), __uint_as_float(r.m[2 * i + 1]));
        v[i] = pack2(__uint_as_float(r.v[2 * i]), __uint_as_float(r.v[2 * i + 1]));
      }
    }
    const float keep = 1.f - a.lr * (o.flags & ADAM_DECAY ? a.wd : 0.f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      m[i] = add2(mul2(both2(a.b1), m[i]), mul2(both2(a.c1), g[i]));
      v[i] = add2(mul2(both2(a.b2), v[i]), mul2(mul2(both2(a.c2), g[i]), g[i]));
      float x, y, d, e; unpack2(v[i], x, y);
      x = adam_root<BITS8>(x); y = adam_root<BITS8>(y);
      root[i] = pack2(x, y);
      unpack2(fma2(root[i], both2(rc2), both2(a.eps)), d, e);
      unpack2(mul2(m[i], both2(lr1)), x, y);
      w[2 * i] = fmaf(__uint_as_float(r.w[2 * i]), keep, -__fdividef(x, d));
      w[2 * i + 1] = fmaf(__uint_as_float(r.w[2 * i + 1]), keep, -__fdividef(y, e));
    }
    if (o.words()) {
      store_words(o.master, reinterpret_cast<const uint32_t (&)[8]>(w));
      if (o.p) *reinterpret_cast<bf16x8*>(o.p) = pack8(w);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) if (e < o.left) {
        o.master[e] = w[e];
        if (o.p) o.p[e] = __float2bfloat16_rn(w[e]);
      }
    }
    const long long s = block * 128 + l16 * 8;
    if (BITS8) {
      uint32_t random[8], bm, bv;
#pragma unroll
      for (int e = 0; e < 8; e++) random[e] = random_bits((uint32_t)s + e, key);
      if (o.left < 8) {                                     // what lies beyond the tensor stays zero
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float x, y;
          unpack2(m[i], x, y); m[i] = pack2(2 * i < o.left ? x : 0.f, 2 * i + 1 < o.left ? y : 0.f);
          unpack2(root[i], x, y); root[i] = pack2(2 * i < o.left ? x : 0.f, 2 * i + 1 < o.left ? y : 0.f);
          unpack2(v[i], x, y); v[i] = pack2(2 * i < o.left ? x : 0.f, 2 * i + 1 < o.left ? y : 0.f);
        }
      }
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.m) + s) = round_block<false>(m, m, random, mask, bm);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.v) + s) = round_block<true>(root, v, random, mask, bv);
      if (l16 == 0) { a.ms[block] = bm; a.vs[block] = bv; }
    } else {
      store_words(static_cast<float*>(a.m) + s, reinterpret_cast<const uint32_t (&)[8]>(m));
      store_words(static_cast<float*>(a.v) + s, reinterpret_cast<const uint32_t (&)[8]>(v));
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
  const long long want = (blocks + 15) / 16, most = 148 * (bits8 ? 3 : 2);
  const unsigned grid = (unsigned)(want < 1 ? 1 : want < most ? want : most);
  const cudaError_t e = launch_pdl(bits8 ? adamw_many_kernel<true> : adamw_many_kernel<false>, dim3(grid), 256, 0, (cudaStream_t)stream, a);
  return e == cudaSuccess ? 0 : (int)e;
}

}  // extern "C"
