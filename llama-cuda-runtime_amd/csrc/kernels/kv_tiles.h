// Operands of the 16x16x32 matrix instructions, and key and value tiles in LDS
// in the layouts attention feeds them from.
#pragma once

#include "device_common.h"

namespace lcr {

#if defined(LCR_ELEM_FP16)
typedef _Float16 mfma_in8 __attribute__((ext_vector_type(8)));
#else
typedef __bf16 mfma_in8 __attribute__((ext_vector_type(8)));
#endif
typedef float mfma_acc4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ mfma_acc4 mfma16x16x32(const mfma_in8& a, const mfma_in8& b,
                                                  const mfma_acc4& c) {
#if defined(LCR_ELEM_FP16)
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
#else
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
#endif
}

__device__ __forceinline__ mfma_in8 as_operand(const vec16& v) {
  return __builtin_bit_cast(mfma_in8, v);
}
__device__ __forceinline__ mfma_in8 lds_operand(const elem_t* p) {
  return *reinterpret_cast<const mfma_in8*>(p);
}

// Two floats rounded to the element type (nearest even) by the packed
// hardware conversion, low half first.
__device__ __forceinline__ uint32_t pack_rounded(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
#if defined(LCR_ELEM_FP16)
  typedef _Float16 e16x2 __attribute__((ext_vector_type(2)));
#else
  typedef __bf16 e16x2 __attribute__((ext_vector_type(2)));
#endif
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, e16x2));
}

// Key rows are head_dim elements with 16-byte chunk c at position
// c ^ key_swizzle(key), so the fragment reads of 16 consecutive keys are free
// of bank conflicts (measured on MI355X for 128-byte rows; 256-byte rows
// spread 16 rows over all 16 chunk positions).
template <int kHeadDim>
__device__ __forceinline__ int key_swizzle(int key) {
  return kHeadDim == 64 ? (key & 7) : (key & 15);
}

// Value rows are kept as they are in the cache (key-major) with chunk c at
// c ^ value_swizzle(key). The P.V operand is assembled by transposing reads
// (ds_read_b64_tr_b16): in each 16-lane group, lane 4k + q names 8 bytes (4
// dims) of one key row and lane 4q + c receives dim c of those 8 bytes from
// the rows named by lanes 4k + q, k = 0..3. One read covers 16 rows x 32
// bytes; with an even swizzle that takes each value twice over the rows of
// one bank half, every bank serves the same number of dwords.
template <int kHeadDim>
__device__ __forceinline__ int value_swizzle(int key) {
  return kHeadDim == 64 ? (key & 6) : ((key & 7) << 1);
}

// The A operand of O^T += V^T . P^T for dims 16 df .. + 15 and the 32 keys
// of half `half` of a value tile (rows of kHeadDim, swizzled as above), in the
// order the P^T fragments hold them: k-slot 8 grp + j is key
// 32 half + 4 grp + j (j < 4) or 32 half + 16 + 4 grp + (j - 4). Two transposing
// reads, one per group of four keys; a lane (16 grp + col) names row
// 4 grp + col / 4 (+ 16) at dims 16 df + 4 (col % 4) .. + 3.
template <int kHeadDim>
__device__ __forceinline__ mfma_in8 transposed_values(const elem_t* tile, int half, int df, int lane) {
  typedef short lds_v4i16 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) lds_v4i16* lds_v4i16_ptr;
  const int col = lane & 15;
  const int grp = lane >> 4;
  const int r0 = 32 * half + 4 * grp + (col >> 2);
  const int c = 2 * df + ((col & 3) >> 1);
  const int within = (col & 1) * 4;
  const int r1 = r0 + 16;
  const elem_t* p0 = tile + r0 * kHeadDim + ((c ^ value_swizzle<kHeadDim>(r0)) << 3) + within;
  const elem_t* p1 = tile + r1 * kHeadDim + ((c ^ value_swizzle<kHeadDim>(r1)) << 3) + within;
  const lds_v4i16 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(p0));
  const lds_v4i16 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_ptr)(p1));
  typedef short v8i16 __attribute__((ext_vector_type(8)));
  const v8i16 both = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(mfma_in8, both);
}

}  // namespace lcr
