// 8-bit codes (e4m3) with an fp32 scale for each block of 128 values:
//   scale = max(max |x|, 2^-100) / 448,  code = e4m3(x * (448 / max(max |x|, 2^-100)))
// 448 is the largest e4m3 value.  The quotients are rounded to fp32 and the product is, before the
// rounding to a code, so a code may be the other neighbour of x / scale where that lies within
// fp32's rounding of the middle of two codes.  The floor keeps the scale of a block of zeros, and
// its reciprocal, finite.  NaN stays NaN and does not count for the maximum; an infinity makes
// its block's scale infinite, and its own code NaN.
#pragma once

#include <cuda_fp8.h>

#include <cstring>
#include <type_traits>

#include "common.cuh"

namespace brt_b200 {

constexpr int kCodeBlock = 128;
constexpr float kCodeMax = 448.f;
constexpr float kAmaxFloor = 7.888609052210118e-31f;  // 2^-100

// Eight neighbouring values of type DT as they lie in memory, 16-byte aligned.
template <int DT>
struct Eight {
  static constexpr int kWords = 8 * (int)sizeof(typename Elem<DT>::type) / 4;
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const typename Elem<DT>::type* p) {
#pragma unroll
    for (int h = 0; h < kWords / 4; h++) {
      const uint4 raw = __ldcs(reinterpret_cast<const uint4*>(p) + h);
      w[4 * h] = raw.x;
      w[4 * h + 1] = raw.y;
      w[4 * h + 2] = raw.z;
      w[4 * h + 3] = raw.w;
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; i++) w[i] = 0u;
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (DT == BRT_F32) {
      return __uint_as_float(w[i]);
    } else {
      const uint16_t bits = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
      typename Elem<DT>::type v;
      memcpy(&v, &bits, 2);
      return Elem<DT>::to_f32(v);
    }
  }
  // The largest magnitude, exact: 16-bit types compare in pairs.  NaN does not count.
  __device__ __forceinline__ float max_abs() const {
    if constexpr (DT == BRT_F32) {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(__uint_as_float(w[i])));
      return m;
    } else {
      using Pair = typename std::conditional<DT == BRT_F16, __half2, __nv_bfloat162>::type;
      Pair m;
      memset(&m, 0, 4);
#pragma unroll
      for (int i = 0; i < kWords; i++) {
        Pair v;
        memcpy(&v, &w[i], 4);
        m = __hmax2(m, __habs2(v));
      }
      return fmaxf(Elem<DT>::to_f32(m.x), Elem<DT>::to_f32(m.y));
    }
  }
  __device__ __forceinline__ uint2 encode(float inverse) const {
    uint32_t c[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(
          make_float2(value(4 * h) * inverse, value(4 * h + 1) * inverse), __NV_SATFINITE,
          __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(
          make_float2(value(4 * h + 2) * inverse, value(4 * h + 3) * inverse), __NV_SATFINITE,
          __NV_E4M3);
      c[h] = lo | hi << 16;
    }
    return make_uint2(c[0], c[1]);
  }
};

}  // namespace brt_b200
