// Values held in 8 bits: codes of float8 e4m3 (finite only: no infinities, 0x7f and 0xff are NaN) or
// int8, to and from float32.
#pragma once
#include "tk_common.hpp"

namespace tk8 {

constexpr int kE4M3 = 0, kInt8 = 1;  // tk_append_quantized and the calls beside it name them so

// The largest magnitude a code holds.
template <int kType>
constexpr float kMost = kType == kE4M3 ? 448.f : 127.f;

typedef float f32x2 __attribute__((ext_vector_type(2)));

// Four values (magnitudes up to kMost, and a rounding above) as codes, rounded to nearest even.
template <int kType>
__device__ __forceinline__ int encode4(const float* x) {
  if constexpr (kType == kE4M3) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], r, true);
  } else {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r |= (uint32_t(int(__builtin_rintf(x[i]))) & 255u) << (8 * i);
    return int(r);
  }
}

// Four codes as float32 (exact).
template <int kType>
__device__ __forceinline__ void decode4(int c, float* x) {
  if constexpr (kType == kE4M3) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(c, false);
    const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
    x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = float(int8_t(uint32_t(c) >> (8 * i)));
  }
}

}  // namespace tk8
