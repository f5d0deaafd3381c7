// 8-bit codes (e4m3) with an fp32 scale for each block of 128 values:
//   scale = max(max |x|, 2^-100) / 448,  code = e4m3(x * (448 / max(max |x|, 2^-100)))
// 448 is the largest e4m3 value.  The quotients are rounded to fp32 and the product is, before the
// rounding to a code, so a code may be the other neighbour of x / scale where that lies within
// fp32's rounding of the middle of two codes.  The floor keeps the scale of a block of zeros, and
// its reciprocal, finite.  NaN stays NaN and does not count for the maximum; an infinity makes
// its block's scale infinite, and its own code NaN.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace brt_b200 {

constexpr int kCodeBlock = 128;
constexpr float kCodeMax = 448.f;
constexpr float kAmaxFloor = 7.888609052210118e-31f;  // 2^-100

// Eight neighbouring values of type DT, 16-byte aligned, as fp32.
template <int DT>
__device__ __forceinline__ void load_eight(const typename Elem<DT>::type* p, float (&v)[8]) {
  using E = Elem<DT>;
  constexpr int kPer = 16 / (int)sizeof(typename E::type);
#pragma unroll
  for (int h = 0; h < 8 / kPer; h++) {
    const uint4 raw = __ldcs(reinterpret_cast<const uint4*>(p + h * kPer));
    typename E::type part[kPer];
    memcpy(part, &raw, 16);
#pragma unroll
    for (int i = 0; i < kPer; i++) v[h * kPer + i] = E::to_f32(part[i]);
  }
}
__device__ __forceinline__ float max_abs(const float (&v)[8]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(v[i]));
  return m;
}
__device__ __forceinline__ uint2 encode_eight(const float (&v)[8], float inverse) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(
        make_float2(v[4 * h] * inverse, v[4 * h + 1] * inverse), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(
        make_float2(v[4 * h + 2] * inverse, v[4 * h + 3] * inverse), __NV_SATFINITE, __NV_E4M3);
    w[h] = lo | hi << 16;
  }
  return make_uint2(w[0], w[1]);
}

}  // namespace brt_b200
