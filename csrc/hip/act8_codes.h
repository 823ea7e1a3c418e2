// act8_codes.h — the 8-bit code of activation checkpoints: a group's power
// of two, and 8 values to and from e4m3 (see act8.hip for the format).
#pragma once

#include "device_types.h"

namespace baguanet {

template <typename T>
struct PowerRange {
  static constexpr int lo = -117, hi = 120;
};
template <>
struct PowerRange<fp16> {
  static constexpr int lo = -15, hi = 8;
};

__device__ inline float power_of_two(int e) {  // -126 <= e <= 127
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

__device__ inline bool is_finite(float v) {
  return fabsf(v) < __builtin_inff();
}

// The power of the group that four neighbouring lanes hold, 8 values each.
template <typename T>
__device__ inline int group_power(float8 v) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < kVec; i++)
    top = fmaxf(top, is_finite(v[i]) ? fabsf(v[i]) : 0.f);
  top = fmaxf(top, __shfl_xor(top, 1));
  top = fmaxf(top, __shfl_xor(top, 2));
  if (top == 0.f) return 0;
  // 448 = 1.75 * 2^8: one power more where the significand passes 1.75
  const uint32_t bits = __float_as_uint(top);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  e = e < PowerRange<T>::lo ? PowerRange<T>::lo : e;
  return e > PowerRange<T>::hi ? PowerRange<T>::hi : e;
}

// 8 codes.  v * 2^-e is exact (or far below the last code's half), so each
// value is rounded once.
template <typename T>
__device__ inline uint2 encode8(float8 v, int e) {
  const float scale = power_of_two(-e);
  const float cap = e == PowerRange<T>::hi ? 240.f : 448.f;
  float w[kVec];
#pragma unroll
  for (int i = 0; i < kVec; i++)
    w[i] = is_finite(v[i]) ? fminf(fmaxf(v[i] * scale, -cap), cap)
                           : __builtin_nanf("");
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(w[0], w[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(w[2], w[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(w[4], w[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(w[6], w[7], hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}

__device__ inline float8 decode8(uint2 q, int e) {
  const float scale = power_of_two(e);
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, false);
  const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, true);
  const auto c = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, false);
  const auto d = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, true);
  float8 v = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  return v * scale;
}

}  // namespace baguanet
