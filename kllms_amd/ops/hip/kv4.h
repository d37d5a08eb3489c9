// Rows of a key/value cache held in 4 bits (head size 128).
//
// 64 neighbouring values are a group: its least value and its step, (most - least) / 15, are bf16 (of bf16 rows the least
// value is one of them, so it is exact), and a value is the whole number of steps above the least one, to the nearest, halves to even:
// at most half a step off, 0.09 of a group's standard deviation where that is normal. A group with a value that is no
// finite number, or whose range is none, is NaN as a whole. The step's own rounding moves the far end of a group by 15 * 2^-9 of a
// step.
//
// 16 words of 32 bits: nibble p of word n is value 32 (p mod 4) + 16 (p div 4) + n. So a lane that has words 4 c.. of a key has
// the values of two 16x16x32 fragments of either group by a mask, and one that has word n of eight keys has column n of each
// of eight 16-column tiles of V. Behind the codes, in a tensor of their own, (step, least) of both groups: 72 bytes a row, bf16 256.
#pragma once

#include "common.h"

#define KV4_BYTES 64       // codes of a row
#define KV4_GROUPS 2       // words of (step, least)

typedef unsigned int u32x2_kv4 __attribute__((ext_vector_type(2)));

struct Kv4Group {
  float step, least, inverse;
  // sound: no value of the group is NaN
  __device__ __forceinline__ Kv4Group(float lo, float hi, bool sound) {
    const float range = hi - lo;
    const bool fine = sound && fabsf(range) < INFINITY;
    step = bf16_to_f32(f32_to_bf16(range / 15.0f));
    step = step >= 1.17549435e-38f ? step : 0.0f;      // a step below the normal numbers is none: its inverse would be infinite
    inverse = step > 0.0f ? 1.0f / step : 0.0f;
    least = fine ? lo : __uint_as_float(0x7fc00000u);
    step = fine ? step : least;
    inverse = fine ? inverse : 0.0f;
  }
  // (x - least) / step as one division rounds it, by the inverse and what it leaves, then to a whole number
  __device__ __forceinline__ uint32_t code(float x) const {
    const float t = x - least, q = t * inverse;
    const float n = __builtin_rintf(__builtin_fmaf(__builtin_fmaf(-q, step, t), inverse, q));
    return (uint32_t)fminf(fmaxf(n, 0.0f), 15.0f);     // NaN: 0
  }
  __device__ __forceinline__ uint32_t word() const {
    return (__float_as_uint(step) >> 16) | (__float_as_uint(least) & 0xffff0000u);
  }
};

__device__ __forceinline__ float kv4_step(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float kv4_least(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// The row of eight neighbouring lanes (aligned), of which the piece-th has values 8 piece.. (a) and 64 + 8 piece.. (b), to
// codes (64 bytes) and scales (2 words).
__device__ __forceinline__ void kv4_store_row(uint32_t* __restrict__ codes, uint32_t* __restrict__ scales, int piece,
                                              const bf16x8_vec& a, const bf16x8_vec& b) {
  float lo[2], hi[2];
  bool nan[2] = {false, false};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    lo[e] = hi[e] = bf16_to_f32(e ? b[0] : a[0]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = bf16_to_f32(e ? b[j] : a[j]);
      lo[e] = fminf(lo[e], x);
      hi[e] = fmaxf(hi[e], x);
      nan[e] |= x != x;
    }
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) {
      lo[e] = fminf(lo[e], __shfl_xor(lo[e], off));
      hi[e] = fmaxf(hi[e], __shfl_xor(hi[e], off));
    }
  }
  const int lane = threadIdx.x & 63, mine = lane & ~7;
  const bool sound[2] = {(__ballot(nan[0]) >> mine & 0xff) == 0, (__ballot(nan[1]) >> mine & 0xff) == 0};
  const Kv4Group ga(lo[0], hi[0], sound[0]), gb(lo[1], hi[1], sound[1]);
  // words 8 (piece & 1) + j: this lane has two of their nibbles, lanes piece ^ 2, ^ 4, ^ 6 the others
  const int at = ((piece >> 2) + 4 * (piece >> 1 & 1)) * 4;
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = (ga.code(bf16_to_f32(a[j])) | gb.code(bf16_to_f32(b[j])) << 8) << at;
  // halves, then quarters of the eight words
  const bool far = piece & 4, next = piece & 2;
  uint32_t h[4], r[2];
#pragma unroll
  for (int j = 0; j < 4; ++j) h[j] = (far ? w[4 + j] : w[j]) | __shfl_xor(far ? w[j] : w[4 + j], 4);
#pragma unroll
  for (int j = 0; j < 2; ++j) r[j] = (next ? h[2 + j] : h[j]) | __shfl_xor(next ? h[j] : h[2 + j], 2);
  *reinterpret_cast<u32x2_kv4*>(codes + 8 * (piece & 1) + (far ? 4 : 0) + (next ? 2 : 0)) = u32x2_kv4{r[0], r[1]};
  if (piece == 0) *reinterpret_cast<u32x2_kv4*>(scales) = u32x2_kv4{ga.word(), gb.word()};
}
