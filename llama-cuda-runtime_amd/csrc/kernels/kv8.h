// The 8-bit cache of lcr_batch.h: its view, its numbers and its scales.
#pragma once

#include "../../../include/lcr_batch.h"
#include "device_common.h"

namespace lcr {

constexpr int kKv8Block = LCR_KV8_BLOCK;

// lcr_kv8_view with its fields' meaning in C++.
struct Kv8View {
  uint8_t* keys;
  uint8_t* values;
  float* key_scales;
  float* value_scales;
  const int32_t* page_table;
  int page_size;
  int page_stride;
  int head_stride;
  int scale_page_stride;
  int scale_head_stride;
  int num_kv_heads;
  int head_dim;

  static Kv8View from_c(const lcr_kv8_view& c) {
    return Kv8View{static_cast<uint8_t*>(c.keys), static_cast<uint8_t*>(c.values), c.key_scales, c.value_scales,
                   c.page_table, c.page_size, c.page_stride, c.head_stride, c.scale_page_stride, c.scale_head_stride,
                   c.num_kv_heads, c.head_dim};
  }

  // First byte of block n of a page's head, and the place of its scale.
  __device__ __forceinline__ size_t block_at(int page, int head, int n) const {
    return static_cast<size_t>(page) * static_cast<size_t>(page_stride) +
           static_cast<size_t>(head) * static_cast<size_t>(head_stride) +
           static_cast<size_t>(n) * static_cast<size_t>(kKv8Block * head_dim);
  }
  __device__ __forceinline__ size_t scale_at(int page, int head, int n) const {
    return static_cast<size_t>(page) * static_cast<size_t>(scale_page_stride) +
           static_cast<size_t>(head) * static_cast<size_t>(scale_head_stride) + static_cast<size_t>(n);
  }
};

// A block's byte of dim i of position t.
__device__ __forceinline__ int kv8_key_byte(int head_dim, int t, int i) { return t * head_dim + i; }
__device__ __forceinline__ int kv8_value_byte(int head_dim, int t, int i) {
  return (t >> 2) * 4 * head_dim + 4 * i + (t & 3);
}

constexpr uint32_t kKv8Nan = 0x7fu;

// The least exponent of a scale, with which the smallest number, 2^-9, still
// stands for a value of the element type (a normal one in bf16), and the largest
// value: 15 / 8 of the type's largest power of two, as the next e4m3 number past it
// is out of the type's range.
#if defined(LCR_ELEM_FP16)
constexpr int kKv8LeastExponent = -15;
constexpr float kKv8Largest = 61440.0f;
#else
constexpr int kKv8LeastExponent = -117;
constexpr float kKv8Largest = 0x1.ep127f;
#endif

__device__ __forceinline__ float power_of_two(int exponent) {
  return __builtin_bit_cast(float, static_cast<uint32_t>(exponent + 127) << 23);
}

// A value as it is held: finite ones within the largest.
__device__ __forceinline__ float kv8_clamped(float v) {
  return fabsf(v) < __builtin_huge_valf() ? __builtin_fminf(__builtin_fmaxf(v, -kKv8Largest), kKv8Largest) : v;
}
// What it counts for a scale: nothing if it is held as NaN.
__device__ __forceinline__ float kv8_size(float clamped) {
  const float a = fabsf(clamped);
  return a < __builtin_huge_valf() ? a : 0.0f;
}

// The exponent of the least power of two with which `largest` (finite, no less than
// 0) is at most 448 = 1.75 * 2^8.
__device__ __forceinline__ int kv8_exponent_for(float largest) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, largest);
  const int exponent = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(exponent, kKv8LeastExponent);
}

// Two values, already divided by their scale (at most 448 in size, or not finite), as
// e4m3 numbers in a word's low two bytes. The conversion rounds to nearest even.
__device__ __forceinline__ uint32_t kv8_pair(float a, float b) {
  uint32_t w = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false)) & 0xffffu;
  if (!(fabsf(a) < __builtin_huge_valf())) w = (w & 0xff00u) | kKv8Nan;
  if (!(fabsf(b) < __builtin_huge_valf())) w = (w & 0x00ffu) | (kKv8Nan << 8);
  return w;
}

__device__ __forceinline__ float kv8_number(uint8_t byte) {
  return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(byte), 0);
}

}  // namespace lcr
