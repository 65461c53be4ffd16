// What the paged KV-cache kernels share: the two 16-bit types, the e4m3
// cache's codes and scales, and cross-lane steps on 64-wide waves.
//
// A quantised cache holds e4m3 codes and, for every token and head, one
// byte s that stands for the scale 2^(s-127) (s = 0: 2^-127, 255: NaN).
// A scale that is a power of two makes x / scale exact, so a code is off
// by its own rounding alone and every reader gets the same value; against
// a free 32-bit scale nothing is lost above e4m3's subnormals, and a row
// of 128 values costs 129 bytes instead of 132.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

namespace paged {

typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));

struct Bf16 {
  typedef __bf16 T;
  typedef __bf16 V2 __attribute__((ext_vector_type(2)));
  typedef __bf16 V8 __attribute__((ext_vector_type(8)));
};

struct Fp16 {
  typedef _Float16 T;
  typedef _Float16 V2 __attribute__((ext_vector_type(2)));
  typedef _Float16 V8 __attribute__((ext_vector_type(8)));
};

// 8 values of 16 bits as they are loaded and stored
template <typename K>
union Oct {
  u4 raw;
  typename K::T h[8];
  typename K::V8 v;
};

__device__ inline float scale_of(uint32_t s) {
  // 2^-127 is a subnormal of its own; 255 has no value
  uint32_t bits = s == 255 ? 0x7fc00000u : s ? s << 23 : 0x00400000u;
  return __uint_as_float(bits);
}

__device__ inline float nan_f32() { return __uint_as_float(0x7fc00000u); }

// the values of 4 codes, times their scale
__device__ inline f4 e4m3_values(uint32_t codes, float scale) {
  f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false);
  f2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
  return f4{lo[0] * scale, lo[1] * scale, hi[0] * scale, hi[1] * scale};
}

__device__ inline uint32_t e4m3_codes(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

}  // namespace paged
