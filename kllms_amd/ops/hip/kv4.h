// Rows of a key/value cache held in 4 bits (head size 128).
//
// 64 neighbouring values are a group: its least value and its step, (most - least) / 15, are bf16 (of bf16 rows the least
// value is one of them, so it is exact), and a value is the whole number of steps above the least one, to the nearest, halves to even:
// at most half a step off, 0.09 of a group's standard deviation where that is normal. A group with a value that is no
// finite number, or whose range is none, is NaN as a whole. The step's own rounding moves the far end of a group by up to 15 * 2^-8 of
// a step.
//
// 16 words of 32 bits: nibble p of word n is value 32 (p mod 4) + 16 (p div 4) + n. So a lane that has words 4 c.. of a key has
// the values of two 16x16x32 fragments of either group by a mask, and one that has word n of eight keys has column n of each
// of eight 16-column tiles of V. Behind the codes, in a tensor of their own, (step, least) of both groups: 72 bytes a row, bf16 256.
#pragma once

#include "common.h"

#define KV4_BYTES 64       // codes of a row
#define KV4_GROUPS 2       // words of (step, least)

typedef unsigned int u32x4_kv4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_kv4 __attribute__((ext_vector_type(2)));

struct Kv4Group {
  float step, least, inverse;
  // sound: no value of the group is NaN; or lo and hi are NaN where one is
  __device__ __forceinline__ Kv4Group(float lo, float hi, bool sound) {
    const float range = hi - lo;
    const bool fine = sound && fabsf(range) < INFINITY;
    // a fifteenth and the inverse as divisions round them, by an estimate and what it leaves
    const float part = range * (1.0f / 15.0f);
    step = bf16_to_f32(f32_to_bf16(__builtin_fmaf(__builtin_fmaf(-part, 15.0f, range), 1.0f / 15.0f, part)));
    step = step >= 1.17549435e-38f ? step : 0.0f;      // a step below the normal numbers is none: its inverse would be infinite
    const float near = __builtin_amdgcn_rcpf(step);
    inverse = step > 0.0f ? __builtin_fmaf(__builtin_fmaf(-near, step, 1.0f), near, near) : 0.0f;
    least = fine ? lo : __uint_as_float(0x7fc00000u);
    step = fine ? step : least;
    inverse = fine ? inverse : 0.0f;
  }
  // (x - least) / step as one division rounds it, by the inverse and what it leaves, to a whole number in the lowest byte: added
  // to 1.5 * 2^23 a small number is rounded to the nearest, halves to even, and stands in the last bits. It is 0 to 15: the
  // step's rounding makes no quotient larger than 15 (1 + 2^-8). Of a group that is not fine the byte is 0: what NaN leaves there.
  __device__ __forceinline__ uint32_t code(float x) const {
    const float t = x - least, q = t * inverse;
    return __float_as_uint(__builtin_fmaf(__builtin_fmaf(-q, step, t), inverse, q) + 12582912.0f);
  }
  __device__ __forceinline__ uint32_t word() const {
    return (__float_as_uint(step) >> 16) | (__float_as_uint(least) & 0xffff0000u);
  }
};

// codes of a value of each group: bytes 0 and 1
__device__ __forceinline__ uint32_t kv4_pair(const Kv4Group& ga, const Kv4Group& gb, float x, float y) {
  return __builtin_amdgcn_perm(gb.code(y), ga.code(x), 0x0c0c0400u);
}

__device__ __forceinline__ float kv4_step(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float kv4_least(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// moves between the eight lanes of a row: ^ 1, ^ 2, ^ 7 (and 3 for ^ 4)
#define KV4_NEXT 0xB1
#define KV4_PAIR 0x4E
#define KV4_BACK 0x141
#define KV4_QUAD 0x1B
template <int HOW>
__device__ __forceinline__ uint32_t kv4_moved(uint32_t x) { return __builtin_amdgcn_update_dpp(x, x, HOW, 0xf, 0xf, true); }

// op over the eight lanes
template <class T, class Op>
__device__ __forceinline__ T kv4_over_row(T x, Op op) {
  x = op(x, __builtin_bit_cast(T, kv4_moved<KV4_NEXT>(__builtin_bit_cast(uint32_t, x))));
  x = op(x, __builtin_bit_cast(T, kv4_moved<KV4_PAIR>(__builtin_bit_cast(uint32_t, x))));
  return op(x, __builtin_bit_cast(T, kv4_moved<KV4_BACK>(__builtin_bit_cast(uint32_t, x))));
}

// The row of eight neighbouring lanes (aligned), of which the piece-th has values 8 piece.. (a) and 64 + 8 piece.. (b), to
// codes (64 bytes) and scales (2 words).
__device__ __forceinline__ void kv4_store_row(uint32_t* __restrict__ codes, uint32_t* __restrict__ scales, int piece,
                                              const bf16x8_vec& a, const bf16x8_vec& b) {
  float lo[2], hi[2];
  // NaN where a value is: the group is none then
  auto least = [](float x, float y) { return __builtin_elementwise_minimum(x, y); };
  auto most = [](float x, float y) { return __builtin_elementwise_maximum(x, y); };
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = bf16_to_f32(e ? b[j] : a[j]);
    lo[e] = least(least(least(x[0], x[1]), least(x[2], x[3])), least(least(x[4], x[5]), least(x[6], x[7])));
    hi[e] = most(most(most(x[0], x[1]), most(x[2], x[3])), most(most(x[4], x[5]), most(x[6], x[7])));
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) lo[e] = kv4_over_row(lo[e], least), hi[e] = kv4_over_row(hi[e], most);
  const Kv4Group ga(lo[0], hi[0], true), gb(lo[1], hi[1], true);
  // words 8 (piece & 1) + j: this lane has two of their nibbles, lanes piece ^ 2, ^ 4, ^ 6 the others
  const int at = ((piece >> 2) + 4 * (piece >> 1 & 1)) * 4;
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    w[j] = kv4_pair(ga, gb, bf16_to_f32(a[j]), bf16_to_f32(b[j])) << at;
  // halves, then quarters of the eight words
  const bool far = piece & 4, next = piece & 2;
  uint32_t h[4], r[2];
#pragma unroll
  for (int j = 0; j < 4; ++j) h[j] = (far ? w[4 + j] : w[j]) | kv4_moved<KV4_QUAD>(kv4_moved<KV4_BACK>(far ? w[j] : w[4 + j]));
#pragma unroll
  for (int j = 0; j < 2; ++j) r[j] = (next ? h[2 + j] : h[j]) | kv4_moved<KV4_PAIR>(next ? h[j] : h[2 + j]);
  *reinterpret_cast<u32x2_kv4*>(codes + 8 * (piece & 1) + (far ? 4 : 0) + (next ? 2 : 0)) = u32x2_kv4{r[0], r[1]};
  if (piece == 0) *reinterpret_cast<u32x2_kv4*>(scales) = u32x2_kv4{ga.word(), gb.word()};
}
