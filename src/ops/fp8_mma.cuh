// The instructions of products in the format of fp8.cuh: tcgen05.mma kind::mxf8f6f4 on a pair of CTAs, and the tensor maps of their operands.
#pragma once
#include "../include/sm100_gemm_pair.cuh"

namespace sm100 {

// Instruction descriptor of kind::mxf8f6f4: e4m3 x e4m3, scales ue8m0, both operands K-major; the byte of the scale words comes on top
__host__ __device__ constexpr uint32_t make_idesc_mxf8(uint32_t M, uint32_t N) { return ((N >> 3) << 17) | (1u << 23) | ((M >> 7) << 27); }
__device__ __forceinline__ uint32_t idesc_bytes(uint32_t a, uint32_t b) { return a << 29 | b << 4; }
// 32 rows of 16 bytes, unswizzled: groups of 8 rows are 128 bytes apart
__device__ __forceinline__ uint64_t make_smem_desc_scales(const void* p) {
  return (uint64_t)((smem_u32(p) & 0x3FFFFu) >> 4) | (uint64_t)(128u >> 4) << 32 | (uint64_t)1 << 46;
}
__device__ __forceinline__ void scales_to_tmem_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void umma_mxf8_pair(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\ttcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n"
               ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}

// [rows, cols] of elements of esz bytes (1: e4m3, 2: bf16, 4: fp32 or words of scales), boxes of box_rows x box_cols; swizzle: of rows of 128 bytes
inline bool fp8_map(CUtensorMap* out, int esz, const void* base, uint64_t rows, uint64_t cols, uint32_t box_rows, uint32_t box_cols, bool swizzle) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const CUtensorMapDataType type = esz == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : esz == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT32;
  cuuint64_t dims[2] = {cols, rows}, strides[1] = {cols * esz};
  cuuint32_t box[2] = {box_cols, box_rows}, estr[2] = {1, 1};
  return fn(out, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace sm100
