// Rows in 8-bit integers: a scale for each, max |x| / 127, and x / scale to the nearest whole number, halves to even.
#pragma once

#include "common.h"

typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// What rows are multiplied with before they are rounded: 127 / most by an inverse and what it leaves, both taken near one
struct Int8Row {
  float up, most, inverse, scale;
  __device__ __forceinline__ explicit Int8Row(uint32_t bits) {       // of the largest magnitude, as bf16
    const float m = __uint_as_float(bits << 16);
    const bool sound = bits < 0x7f80u;                               // neither infinite nor NaN
    const int e = max((int)(bits >> 7) - 127, -120);
    const float f = ldexpf(1.0f, -e);
    up = 127.0f * f;
    most = m * f;
    inverse = sound && m > 0.0f ? 1.0f / most : 0.0f;
    scale = sound ? m / 127.0f : __uint_as_float(0x7fc00000u);       // such a row is NaN as a whole
  }
  // its code is the lowest byte: added to 1.5 * 2^23, a number this small is rounded as rint does and stands in the last bits. No
  // number passes 127 by as much as that sees; of a row that is not sound the codes do not matter.
  __device__ __forceinline__ uint32_t code(float x) const {
    const float t = x * up, q = t * inverse;
    return __float_as_uint(__builtin_fmaf(__builtin_fmaf(-q, most, t), inverse, q) + 12582912.0f);
  }
  __device__ __forceinline__ uint32_t four(short a, short b, short c, short d) const {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(code(bf16_to_f32(d)), code(bf16_to_f32(c)), 0x0c0c0400u),
                                 __builtin_amdgcn_perm(code(bf16_to_f32(b)), code(bf16_to_f32(a)), 0x0c0c0400u), 0x05040100u);
  }
  __device__ __forceinline__ u32x2 codes(const u16x8& x) const {
    return u32x2{four((short)x[0], (short)x[1], (short)x[2], (short)x[3]), four((short)x[4], (short)x[5], (short)x[6], (short)x[7])};
  }
};
