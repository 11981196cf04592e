// Codes of the paged 8-bit cache: e4m3 (HELD 0) and int8 (HELD 1), four to a word.
#pragma once
#include <hip/hip_runtime.h>

typedef float fx_f32x2 __attribute__((ext_vector_type(2)));

// (the conversion in hardware is the format's own: round to nearest, ties to even, with subnormals; x is held to the largest code
// first, and NaN, which a clamp would take for a bound, is put back)
template <int HELD>
__device__ __forceinline__ unsigned encode4(const float* x) {
  if constexpr (HELD == 0) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = x[i] != x[i] ? x[i] : fminf(fmaxf(x[i], -448.0f), 448.0f);
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
  } else {
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = x[i] != x[i] ? 0.0f : fminf(fmaxf(__builtin_rintf(x[i]), -127.0f), 127.0f);
      w |= ((unsigned)(int)y & 0xffu) << (8 * i);
    }
    return w;
  }
}
template <int HELD>
__device__ __forceinline__ void decode4(float* x, unsigned w) {
  if constexpr (HELD == 0) {
    const fx_f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(signed char)(w >> (8 * i));
  }
}
// The scale of numbers up to `top`: 448 = 1.75 * 2^8 and 127 = 1.984375 * 2^6, so the mantissa of `top` says which power it needs
template <int HELD>
__device__ __forceinline__ float scale_of(float top) {
  constexpr unsigned kMantissa = HELD == 0 ? 0x600000u : 0x7e0000u;
  constexpr int kShift = HELD == 0 ? 8 : 6, kLeast = -100, kMost = HELD == 0 ? 119 : 121;
  const unsigned u = __float_as_uint(top);
  int e = (int)(u >> 23) - 127 - kShift + ((u & 0x7fffffu) > kMantissa ? 1 : 0);   // (zero and subnormals: far below the least)
  e = e < kLeast ? kLeast : e > kMost ? kMost : e;
  return __uint_as_float((unsigned)(e + 127) << 23);
}
