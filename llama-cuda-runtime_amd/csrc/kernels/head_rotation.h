// RMSNorm over a head and its half-split rotation, as lcr_batch.h defines them: what
// the entries that write a step's keys and values have in common.
#pragma once

#include "device_common.h"

namespace lcr {

// Sum over the kLanes lanes (a power of two) that share a head.
template <int kLanes>
__device__ __forceinline__ float head_sum(float v) {
  if constexpr (kLanes >= 16) v += xor_lane<8>(v);
  if constexpr (kLanes >= 8) v += xor_lane<4>(v);
  if constexpr (kLanes >= 4) v += xor_lane<2>(v);
  return v + xor_lane<1>(v);
}

// Elements i .. i + 7 of both halves of a head that kHeadDim / 16 lanes share, in
// place: normed where there is a weight, rotated by the angles of its position.
template <int kHeadDim>
__device__ __forceinline__ void norm_rotate(vec16& lo, vec16& hi, const elem_t* weight, float eps, const float2* angles,
                                            int i) {
  constexpr int kHalf = kHeadDim / 2;
  const float4* cs = reinterpret_cast<const float4*>(angles + i);
  float4 angle[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) angle[j] = cs[j];
  float x[8], y[8];
  unpack8(lo, x);
  unpack8(hi, y);
  if (weight != nullptr) {
    float wx[8], wy[8];
    unpack8(load16(weight + i), wx);
    unpack8(load16(weight + kHalf + i), wy);
    float square = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) square = __builtin_fmaf(x[j], x[j], __builtin_fmaf(y[j], y[j], square));
    const float scale = 1.0f / sqrtf(head_sum<kHeadDim / 16>(square) * (1.0f / kHeadDim) + eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = x[j] * scale * wx[j];
      y[j] = y[j] * scale * wy[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 r0 = rope_rotate(x[2 * j], y[2 * j], make_float2(angle[j].x, angle[j].y));
    const float2 r1 = rope_rotate(x[2 * j + 1], y[2 * j + 1], make_float2(angle[j].z, angle[j].w));
    lo.w[j] = pack_elems(r0.x, r1.x);
    hi.w[j] = pack_elems(r0.y, r1.y);
  }
}

}  // namespace lcr
