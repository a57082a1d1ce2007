// AdamW over many tensors in one launch, moments in fp32 or in 8 bits.
//
//   g' = g * gscale     m' = b1 m + (1 - b1) g'     v' = b2 v + (1 - b2) g' g'     w' = w (1 - lr wd) - lr (m' / (1 - b1^t)) / (sqrt(v' / (1 - b2^t)) + eps)
//
// In 8 bits the moments lie as e4m3 with a power of two for each block of 128 elements (fp8.cuh), the second one as its root: a root has half the range (e4m3's smallest step is
// 2^-18 of a block's largest value, 2^-36 of the largest v) and is what the update divides by.  Both are rounded stochastically, up with the probability of the part cut off.
// Rounded to nearest they would stand still: with b2 = 0.999 a root changes by 0.05 % a step, and e4m3's half step is 3 to 6 %.  A root that is not zero does not become zero, or the
// update of an element whose gradients are 2^-18 of its block's largest would divide by eps alone.  The random bits are a hash of the element's place, the step and a seed, so a run can be
// repeated bit by bit; for the same reason the state's arithmetic is in single roundings (no fma: sum2_alone).  A root that is right in the mean has a square that is too large by the rounding's variance: v by 2.5 to 3.4 %,
// at most 13.5 %.
#include "fp8.cuh"

namespace piccl_ops {

// A tensor: addresses, elements, its first block of 128 in the state, what it is.  Mirrored in piccl_b200/ops/optimizer.py.
struct AdamTensor {
  void* p; float* master; const void* g;
  long long n, block;
  int flags, pad;
};
enum { ADAM_DECAY = 1, ADAM_P_F32 = 2, ADAM_G_F32 = 4, ADAM_WORDS = 8 };      // WORDS: every address on a boundary of eight elements

struct AdamArgs {
  const AdamTensor* tensors; const int* owner; long long blocks;      // owner: the tensor of each block
  void *m, *v; uint8_t *ms, *vs;
  float lr, b1, c1, b2, c2, eps, wd, lb1, lb2;      // c: 1 - b; lb: logarithms
  float gscale, one; const float* gscale_dev;      // one: 1
  int* step; unsigned* ticket; uint32_t seed;
};

// a + b where a is a product that has been rounded.  The compiler makes one fma of a packed product and a packed sum, whatever their rounding modes say (mul.rn.f32x2, add.rn.f32x2); of a product and
// an fma by a factor that it does not know it cannot.
__device__ __forceinline__ f32x2 sum2_alone(f32x2 a, f32x2 b, float one) { return fma2(a, both2(one), b); }

// A function of place and step by their sum: an element's bits are independent from step to step, and those of its neighbour one step apart.
__device__ __forceinline__ uint32_t random_bits(uint32_t place, uint32_t key) {
  uint32_t h = place * 0x9E3779B9u + key;      // the golden ratio, then the roots of 3 and 2: odd numbers without a pattern
  h = (h ^ (h >> 16)) * 0xBB67AE85u;
  return (h ^ (h >> 15)) * 0x6A09E667u;
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
// An element's 16 random bits, of h ^ (h >> 16): the upper half for the root, the lower one for m
template <bool ROOT> __device__ __forceinline__ uint32_t random_part(uint32_t h) { return ROOT ? h >> 16 : (h ^ h >> 16) & 0xffffu; }
// x / scale, at most 448 in magnitude, rounded: what is cut off of its fraction, and the random bits, carry.  Its magnitude is 2^-6 or more: the steps of e4m3 are those of three bits of fraction.
template <bool ROOT> __device__ __forceinline__ float stochastic(float t, uint32_t r) { return __uint_as_float((__float_as_uint(t) + (random_part<ROOT>(r) << 4)) & 0xfff00000u); }
// The same for any magnitude, and NaN for x that is not finite; a root that is not zero stays so.  sum: whose upper bits are taken
template <bool ROOT> __device__ __forceinline__ float stochastic_any(float x, float t, uint32_t r, uint32_t& sum) {
  const float a = fabsf(t), low = a < 0.015625f ? 0.015625f : 0.f;      // below 2^-6 the steps are those of [2^-6, 2^-5)
  sum = __float_as_uint(a + low) + (random_part<ROOT>(r) << 4);
  float z = __uint_as_float(sum & 0xfff00000u) - low;
  if (ROOT && a > 0.f) z = fmaxf(z, 0.001953125f);
  return (__float_as_uint(x) & 0x7fffffffu) >= kInf ? __uint_as_float(0x7fffffffu) : copysignf(z, t);
}
// The byte of a block whose largest value is the root of v: the smallest s for which v <= (448 * 2^s)^2 = 1.53125 * 2^(17 + 2 s).  (A root rounded to fp32 is above 448 * 2^s exactly
// where v is above that, so this is the byte of correctly rounded roots.)
__device__ __forceinline__ uint32_t scale_byte_of_root(uint32_t v_bits) {
  if (v_bits < 0x00800000u) return scale_byte(__float_as_uint(__fsqrt_rn(__uint_as_float(v_bits))));      // the exponent of a v below 2^-126 is not in its bits
  const int e = (int)((v_bits + (0x7fffffu - 0x440000u)) >> 23) - 127 - 17;
  return (uint32_t)(127 + ((e + 1) >> 1));
}
__device__ __forceinline__ uint2 e4m3_bytes(const float (&t)[8]) {
  return make_uint2(e4m3_four(t[0], t[1], t[2], t[3]), e4m3_four(t[4], t[5], t[6], t[7]));
}
// Eight moments and roots of a block, by 16 lanes -> their bytes and the block's two.  All lanes of a warp call it together (votes and shuffles among a part of them cost a barrier each), and both
// maxima are found side by side: one after the other, each behind its own votes, the latencies of shuffles were a third of the kernel's time.
// What is held is the correctly rounded root's: whether the random bits carry can hang on its last bit, and a carry is a whole step of e4m3.  r2 are approximate roots, off by less than four units in the last place (2^-23 is
// two, and half a one is the rounding), so they decide where the sum is at least that far from a carry.  The nearer ones, eight in 2^20, are rounded again from roots by __fsqrt_rn: GPT-2 medium 1178 us, the smallest
// model 8.5 (1137 and 8.5 with approximate roots alone; 1202 and 9.4 with __fsqrt_rn for whatever is below 2^-6 too; 1220 and 9.2 with it throughout).
__device__ __forceinline__ void round_moments(const f32x2 (&m2)[4], const f32x2 (&v2)[4], const f32x2 (&r2)[4], float r_least, uint32_t place, uint32_t key, uint2& m_out, uint2& v_out, uint32_t& m_byte, uint32_t& v_byte) {
  float m[8], v[8];
#pragma unroll
  for (int i = 0; i < 4; i++) { unpack2(m2[i], m[2 * i], m[2 * i + 1]); unpack2(v2[i], v[2 * i], v[2 * i + 1]); }
  float m_most = fabsf(m[0]), m_least = fabsf(m[0]), v_most = v[0];
#pragma unroll
  for (int e = 1; e < 8; e += 2) {
    m_most = max3_nan(m_most, fabsf(m[e]), fabsf(m[(e + 1) % 8])); m_least = min3(m_least, fabsf(m[e]), fabsf(m[(e + 1) % 8]));
    v_most = max3_nan(v_most, v[e], v[(e + 1) % 8]);
  }
  uint32_t m_top = __float_as_uint(m_most), v_top = __float_as_uint(v_most);
  bool odd = __any_sync(0xffffffffu, max(m_top, v_top) >= kInf);
  if (odd) {
    m_top = v_top = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) { m_top = max(m_top, finite_bits(m[e])); v_top = max(v_top, finite_bits(v[e])); }
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    const uint32_t x = __shfl_xor_sync(0xffffffffu, m_top, o), y = __shfl_xor_sync(0xffffffffu, v_top, o);
    m_top = max(m_top, x); v_top = max(v_top, y);
  }
  m_byte = scale_byte(m_top); v_byte = scale_byte_of_root(v_top);
  const float fm = scale_inverse(m_byte), fr = scale_inverse(v_byte);
  uint32_t random[8];
#pragma unroll
  for (int e = 0; e < 8; e++) random[e] = random_bits(place + e, key);
  odd = __any_sync(0xffffffffu, odd || fminf(m_least * fm, r_least * fr) < 0.015625f);
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 4; i++) { unpack2(mul2(m2[i], both2(fm)), a[2 * i], a[2 * i + 1]); unpack2(mul2(r2[i], both2(fr)), b[2 * i], b[2 * i + 1]); }
  uint32_t sum[8];                                          // of roots and random bits: the low 20 are cut off
  if (odd) {
#pragma unroll
    for (int e = 0; e < 8; e++) { uint32_t none; a[e] = stochastic_any<false>(m[e], a[e], random[e], none); b[e] = stochastic_any<true>(v[e], b[e], random[e], sum[e]); }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      a[e] = stochastic<false>(a[e], random[e]);
      sum[e] = __float_as_uint(b[e]) + (random_part<true>(random[e]) << 4);
      b[e] = __uint_as_float(sum[e] & 0xfff00000u);
    }
  }
  uint32_t near = 0xffffffffu;
#pragma unroll
  for (int e = 0; e < 8; e += 2) near = __vimin3_u32(near, (sum[e] << 12) + (4u << 12), (sum[e + 1] << 12) + (4u << 12));
  if (__any_sync(0xffffffffu, near < 8u << 12)) {
    asm volatile("" : "+r"(place));                         // the bits are computed again, not kept
#pragma unroll
    for (int e = 0; e < 8; e++) { const float root = __fsqrt_rn(v[e]); uint32_t none; b[e] = stochastic_any<true>(root, root * fr, random_bits(place + e, key), none); }
  }
  m_out = e4m3_bytes(a); v_out = e4m3_bytes(b);
}

// The tensor that a lane works on
struct AdamNow {
  bf16* p; float* master; const void* g;                   // p: null if the parameters are the masters
  long long n, first, end;                                 // elements; its first block, that of the next tensor
  int flags;
};
// N words of 4 bytes from N * 4 bytes' boundary on.  Eight of them in one access of 32 bytes: as two of 16 a warp would touch every sector twice.
template <int N> __device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[N]) {
  static_assert(N == 2 || N == 4 || N == 8, "");
  if constexpr (N == 2) { const uint2 a = *static_cast<const uint2*>(p); w[0] = a.x; w[1] = a.y; }
  else if constexpr (N == 4) { const uint4 a = *static_cast<const uint4*>(p); w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; }
  else asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p) : "memory");
}
template <int N> __device__ __forceinline__ void store_words(void* p, const uint32_t (&w)[N]) {
  static_assert(N == 2 || N == 4 || N == 8, "");
  if constexpr (N == 2) *static_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else if constexpr (N == 4) *static_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
// The tensor of a block.  (By bisection it took eight loads, each waiting for the one before, at almost every block of a thread: a grid is some tensors wide.)
__device__ __forceinline__ void adam_find(const AdamArgs& a, long long block, AdamNow& c) {
  const AdamTensor& q = a.tensors[a.owner[block]];
  c.flags = q.flags; c.g = q.g; c.n = q.n; c.first = q.block;
  c.p = q.flags & ADAM_P_F32 ? nullptr : static_cast<bf16*>(q.p); c.master = q.flags & ADAM_P_F32 ? static_cast<float*>(q.p) : q.master;
  c.end = q.block + (q.n + 127) / 128;
}
// The root of v that the update divides by: in 8 bits the approximate one (to 2^-23, less than the division's own two units; zero for v below 2^-126, which the caller looks after)
template <bool BITS8> __device__ __forceinline__ float adam_root(float v) {
  float r;
  if (BITS8) asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); else r = __fsqrt_rn(v);
  return r;
}
// x / y to two units in the last place: of the change of a weight, which is rounded beside the weight (an exact quotient is a branch and some ten instructions for each element)
__device__ __forceinline__ float div_approx(float x, float y) { float r; asm("div.approx.ftz.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y)); return r; }

// What the step is, for every thread of a block.
// (Every thread computes it for itself while its first loads are under way: through shared memory they would wait for a barrier, a microsecond of a small step's ten.)
struct AdamStep {
  float rc2, lr1, gscale; uint32_t key;
  __device__ __forceinline__ AdamStep(const AdamArgs& a) {
    const int t = *(volatile int*)a.step + 1;
    lr1 = a.lr / -expm1f((float)t * a.lb1);                 // 1 - b^t without cancellation
    rc2 = 1.f / sqrtf(-expm1f((float)t * a.lb2));
    gscale = a.gscale_dev ? a.gscale * *a.gscale_dev : a.gscale;
    key = a.seed + (uint32_t)t * 0x9E3779B9u;
  }
  __device__ __forceinline__ static void done(const AdamArgs& a) {
    __syncthreads();                                       // every thread has read *step
    if (threadIdx.x == 0 && atomicAdd(a.ticket, 1u) == gridDim.x - 1) { *a.ticket = 0; atomicAdd(a.step, 1); }
  }
  // moments, roots and weights of E elements; w: as bits; least: in 8 bits, of the roots
  template <bool BITS8, int E> __device__ __forceinline__ void update(const AdamArgs& a, int flags, const uint32_t (&gw)[E], uint32_t (&w)[E], f32x2 (&m)[E / 2], f32x2 (&v)[E / 2], f32x2 (&root)[E / 2], float& least) const {
    const float keep = 1.f - a.lr * (flags & ADAM_DECAY ? a.wd : 0.f);
#pragma unroll
    for (int k = 0; k < E / 2; k++) {
      f32x2 g = flags & ADAM_G_F32 ? pack2(__uint_as_float(gw[2 * k]), __uint_as_float(gw[2 * k + 1])) : pack2(__uint_as_float(gw[k] << 16), __uint_as_float(gw[k] & 0xffff0000u));
      g = mul2(g, both2(gscale));
      m[k] = sum2_alone(mul2(both2(a.b1), m[k]), mul2(both2(a.c1), g), a.one);
      v[k] = sum2_alone(mul2(both2(a.b2), v[k]), mul2(mul2(both2(a.c2), g), g), a.one);
      float x, y; unpack2(v[k], x, y);
      x = adam_root<BITS8>(x); y = adam_root<BITS8>(y);
      if (BITS8) least = k ? min3(least, x, y) : fminf(x, y);
      root[k] = pack2(x, y);
    }
    if (BITS8 && least == 0.f) {                            // v is zero, or below 2^-126: the root of it times 2^64
#pragma unroll
      for (int k = 0; k < E / 2; k++) {
        float x, y, p, q; unpack2(v[k], x, y); unpack2(root[k], p, q);
        root[k] = pack2(p == 0.f ? adam_root<true>(x * 0x1p64f) * 0x1p-32f : p, q == 0.f ? adam_root<true>(y * 0x1p64f) * 0x1p-32f : q);
      }
    }
#pragma unroll
    for (int k = 0; k < E / 2; k++) {
      float x, y, d, e;
      unpack2(fma2(root[k], both2(rc2), both2(a.eps)), d, e);
      unpack2(mul2(m[k], both2(lr1)), x, y);
      w[2 * k] = __float_as_uint(fmaf(__uint_as_float(w[2 * k]), keep, -div_approx(x, d)));
      w[2 * k + 1] = __float_as_uint(fmaf(__uint_as_float(w[2 * k + 1]), keep, -div_approx(y, e)));
    }
  }
};
// E gradients (bf16 in pairs) and weights one by one; left: how many there are
template <int E> __device__ __forceinline__ void load_some(const void* g, const float* master, int left, int flags, uint32_t (&gw)[E], uint32_t (&w)[E]) {
#pragma unroll
  for (int e = 0; e < E; e++) { gw[e] = 0; w[e] = 0; }
#pragma unroll
  for (int e = 0; e < E; e++) if (e < left) {
    if (flags & ADAM_G_F32) gw[e] = static_cast<const uint32_t*>(g)[e];
    else gw[e >> 1] |= (uint32_t)static_cast<const uint16_t*>(g)[e] << (16 * (e & 1));
    w[e] = __float_as_uint(master[e]);
  }
}
template <int E> __device__ __forceinline__ void store_weights(float* master, bf16* p, int left, bool words, const uint32_t (&w)[E]) {
  if (words) {
    store_words(master, w);
    if (p) {
      uint32_t o[E / 2];
#pragma unroll
      for (int k = 0; k < E / 2; k++) { const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1])); o[k] = *reinterpret_cast<const uint32_t*>(&h); }
      store_words(p, o);
    }
  } else
#pragma unroll
    for (int e = 0; e < E; e++) if (e < left) {
      master[e] = __uint_as_float(w[e]);
      if (p) p[e] = __float2bfloat16_rn(__uint_as_float(w[e]));
    }
}
// What lies beyond a tensor stays zero, whatever the gradients are multiplied by
__device__ __forceinline__ void zero_beyond(int left, f32x2 (&z)[4]) {
#pragma unroll
  for (int k = 0; k < 4; k++) {
    float x, y; unpack2(z[k], x, y);
    z[k] = pack2(2 * k < left ? x : 0.f, 2 * k + 1 < left ? y : 0.f);
  }
}
__device__ __forceinline__ const void* gradients(const AdamNow& c, long long i) { return static_cast<const char*>(c.g) + i * (c.flags & ADAM_G_F32 ? 4 : 2); }

// Moments in fp32: a lane has eight elements, sixteen lanes a block.  Bound by memory: 28 bytes an element (bf16 parameters and gradients, masters).  GPT-2 medium's 355 M parameters: 1570 us, 6.3 TB/s; with four
// elements a lane and 40 warps to an SM in place of 24 it took 1820, with the next block's lines prefetched 1690.
__global__ void __launch_bounds__(256, 3) adamw_many_kernel(const AdamArgs a) {
  constexpr int E = 8;
  pdl_begin();
  const AdamStep step(a);
  const int l = threadIdx.x & 15;
  const long long stride = gridDim.x * 16ll;
  AdamNow now = {nullptr, nullptr, nullptr, 0, 0, -1, 0};
  for (long long block = blockIdx.x * 16ll + (threadIdx.x >> 4); block < a.blocks; block += stride) {
    if (block >= now.end) adam_find(a, block, now);
    const long long i = (block - now.first) * 128 + l * E, s = block * 128 + l * E;
    const int left = (int)min((long long)E, now.n - i);    // elements of this lane (not positive: none)
    const bool words = (now.flags & ADAM_WORDS) && left == E;
    uint32_t gw[E], w[E];
    f32x2 m[4], v[4], root[4];
    load_words(static_cast<const float*>(a.m) + s, reinterpret_cast<uint32_t (&)[E]>(m));
    load_words(static_cast<const float*>(a.v) + s, reinterpret_cast<uint32_t (&)[E]>(v));
    if (words) {
      load_words(now.master + i, w);
      if (now.flags & ADAM_G_F32) load_words(gradients(now, i), gw); else load_words(gradients(now, i), reinterpret_cast<uint32_t (&)[E / 2]>(gw));
    } else load_some(gradients(now, i), now.master + i, left, now.flags, gw, w);
    float unused;
    step.update<false>(a, now.flags, gw, w, m, v, root, unused);
    store_weights(now.master + i, now.p ? now.p + i : nullptr, left, words, w);
    if (left < E) { zero_beyond(left, m); zero_beyond(left, v); }
    store_words(static_cast<float*>(a.m) + s, reinterpret_cast<const uint32_t (&)[E]>(m));
    store_words(static_cast<float*>(a.v) + s, reinterpret_cast<const uint32_t (&)[E]>(v));
  }
  AdamStep::done(a);
}

// Moments in 8 bits: a lane has eight elements, sixteen lanes a block, a warp two blocks.  16 bytes an element (868 us of memory for GPT-2 medium) and about as much arithmetic: two roundings, a root and a division each.
// 1178 us there, 4.8 TB/s.  Of a form before (1115 us): without the prefetch of the next block's lines 1245, with 16 warps to an SM in place of 24 1395.
__global__ void __launch_bounds__(256, 3) adamw_many8_kernel(const AdamArgs a) {
  constexpr int E = 8;
  pdl_begin();
  const AdamStep step(a);
  const int l = threadIdx.x & 15, second = threadIdx.x >> 4 & 1;
  const long long stride = gridDim.x * 16ll;
  AdamNow now = {nullptr, nullptr, nullptr, 0, 0, -1, 0};
  for (long long block = blockIdx.x * 16ll + (threadIdx.x >> 4); block - second < a.blocks; block += stride) {
    const bool there = block < a.blocks;                    // the first half of a warp may have the last block
    if (there && block >= now.end) adam_find(a, block, now);
    const long long i = (block - now.first) * 128 + l * E, s = block * 128 + l * E;
    const int left = there ? (int)min((long long)E, now.n - i) : 0;
    const bool words = (now.flags & ADAM_WORDS) && left == E;
    uint32_t gw[E], w[E], mw[2] = {0, 0}, vw[2] = {0, 0}, mb = 0, vb = 0;
    if (there) {
      load_words(static_cast<const uint8_t*>(a.m) + s, mw);
      load_words(static_cast<const uint8_t*>(a.v) + s, vw);
      mb = a.ms[block]; vb = a.vs[block];
    }
    if (words) {
      load_words(now.master + i, w);
      if (now.flags & ADAM_G_F32) load_words(gradients(now, i), gw); else load_words(gradients(now, i), reinterpret_cast<uint32_t (&)[E / 2]>(gw));
    } else load_some(gradients(now, i), now.master + i, left, now.flags, gw, w);
    const long long next = block + stride, j = (next - now.first) * 128;
    if (j + 128 <= now.n && l < 8) {                        // the next block, if it is a whole one of this tensor, on its way into L2: a line of 128 bytes a lane
      const char* const at = l < 4 ? reinterpret_cast<const char*>(now.master + j) + l * 128 : l < 6 ? static_cast<const char*>(gradients(now, j)) + (l - 4) * 128
                             : (l == 6 ? static_cast<const char*>(a.m) : static_cast<const char*>(a.v)) + next * 128;
      asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
    }
    f32x2 m[4], v[4], root[4];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      e4m3_values(mw[k], scale_value(mb), reinterpret_cast<f32x2 (&)[2]>(m[2 * k]));
      e4m3_values(vw[k], scale_value(vb), reinterpret_cast<f32x2 (&)[2]>(v[2 * k]));
    }
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = mul2(v[k], v[k]);
    float least;                                            // of the roots
    step.update<true>(a, now.flags, gw, w, m, v, root, least);
    store_weights(now.master + i, now.p ? now.p + i : nullptr, left, words, w);
    if (left < E) { zero_beyond(left, m); zero_beyond(left, root); zero_beyond(left, v); }
    uint2 om, ov;
    round_moments(m, v, root, least, (uint32_t)s, step.key, om, ov, mb, vb);
    if (!there) continue;
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.m) + s) = om;
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.v) + s) = ov;
    if (l == 0) { a.ms[block] = mb; a.vs[block] = vb; }
  }
  AdamStep::done(a);
}

}  // namespace piccl_ops

using namespace piccl_ops;

extern "C" {

// tensors: device array of records in the order of their blocks, which follow each other and cover [0, blocks), none of them empty; owner: device ints, the record of each block; m, v: blocks * 128 elements (fp32, or bytes with a byte of scale for each
// block); step: device int, steps done so far, advanced by the launch; ticket: device int that holds zero.  gscale_dev: null, or a device float that multiplies gscale.
int piccl_ops_adamw_many(const void* tensors, const int* owner, long long blocks, int bits8, void* m, void* v, void* ms, void* vs, float lr, double b1, double b2, float eps, float wd, float gscale,
                         const float* gscale_dev, int* step, unsigned* ticket, unsigned seed, void* stream) {
  if (blocks < 0 || !(b1 >= 0 && b1 < 1) || !(b2 >= 0 && b2 < 1)) return -1;
  if ((blocks && (!tensors || !owner || !m || !v || (bits8 && (!ms || !vs)))) || !step || !ticket) return -2;
  if ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v)) & 31) return -2;      // the kernel's accesses of 32 bytes
  AdamArgs a{static_cast<const AdamTensor*>(tensors), owner, blocks, m, v, (uint8_t*)ms, (uint8_t*)vs, lr, (float)b1, (float)(1 - b1), (float)b2, (float)(1 - b2), eps, wd, (float)log(b1), (float)log(b2),
             gscale, 1.f, gscale_dev, step, ticket, seed};
  const long long want = (blocks + 15) / 16, most = 148 * 3;
  const dim3 grid((unsigned)(want < 1 ? 1 : want < most ? want : most));
  const cudaError_t e = launch_pdl(bits8 ? adamw_many8_kernel : adamw_many_kernel, grid, 256, 0, (cudaStream_t)stream, a);
  return e == cudaSuccess ? 0 : (int)e;
}

}  // extern "C"
