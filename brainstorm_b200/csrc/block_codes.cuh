// 8-bit codes (e4m3) with an fp32 scale for each block of 128 values:
//   scale = max(max |x|, 2^-100) / 448,  code = e4m3(x / scale)
// 448 is the largest e4m3 value.  Both quotients are rounded to fp32 as IEEE division does: values
// that lie in the middle of two codes are common (bf16 inputs whose maximum is a multiple of 7),
// and a product with a rounded reciprocal sends them to either side.  Where max / 448 itself is
// rounded, a value in the middle of two codes by the unrounded quotient may lie 2^-24 beside it and
// goes to that side: 8 in 10000 codes of bf16 values then are the other one of two codes equally near.
// The floor keeps the scale of a block of zeros, and its reciprocal, finite.  NaN stays NaN and does
// not count for the maximum; an infinity makes its block's scale infinite and its codes NaN.
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
    } else if constexpr (DT == BRT_BF16) {
      return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
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
  // value / scale for all eight, from an approximate reciprocal, by Markstein's last step of a
  // division: the remainder of the first quotient is exact, and adding its own quotient rounds
  // correctly.
  __device__ __forceinline__ uint2 encode(float scale, float inverse) const {
    const float2 inv = make_float2(inverse, inverse), minus = make_float2(-scale, -scale);
    uint32_t pair[4];
#pragma unroll
    for (int h = 0; h < 4; h++) {
      const float2 v = make_float2(value(2 * h), value(2 * h + 1));
      const float2 first = __fmul2_rn(v, inv);
      const float2 rest = __ffma2_rn(first, minus, v);
      pair[h] = __nv_cvt_float2_to_fp8x2(__ffma2_rn(rest, inv, first), __NV_SATFINITE, __NV_E4M3);
    }
    return make_uint2(pair[0] | pair[1] << 16, pair[2] | pair[3] << 16);
  }
};

}  // namespace brt_b200
