// Attention of prompt portions (rows behind a cached prefix, causal among themselves) against a paged cache held in 4 bits
// (kv4.h), for gfx950.
//
//   - an 8-wave workgroup serves 32-row tiles of all query heads of ONE kv head of a segment: 256 / GQA rows, a wave for
//     each tile and head. So the keys are made once for all heads, and a short tail still has eight waves at work
//   - 128 keys at a time: each thread has a quarter of a K row and of a V row on their way in registers, makes fp16 of them
//     and puts them to LDS, double-buffered, while the stage before is multiplied
//   - fp16 holds what the cache stands for to 2^-11 (with K in bf16 the result is three times further off than its own
//     rounding makes it, behind 9000 keys). Of a group whose largest is not between 2^-10 and 2^14 a power of 2^16 is taken out that
//     brings it there: none, in a model, and then nothing is multiplied back. Each group has its own: with one for both of a row, values 2^-20
//     of the other group's were up to 16 % off. q's rows are scaled into fp16's range exactly
//   - scores and softmax as in attn_prefill.hip: S = K Q^T, a lane has one row's scores, base-2 exponentials of one fma, the
//     running max renewed when it grows by more than 8; P is fp16 in one part, 2^-11 of it, where bf16 would need two. Below 2^-14 of
//     the running max it is off by 2^-25 of that, as much as a sum in fp32 loses of it
//   - few or long groups are cut along the keys (the plan says where); their sums meet in a second launch
//
// A nibble becomes fp16 in three half instructions of two each: masked into 1024 + n, less 1024, times step plus least
// value, which is rounded once.
//
// What bounds it: the vector units, with the softmax's exponentials before all; making the keys is a sixth of their work. The two
// waves of a SIMD do not cover one's products by the other's exponentials for long: they meet at each stage's barrier (vector
// instructions 59 % of a SIMD's time, matrix instructions 39 %, so hardly at once); that one half of
// them loads before its products and the other half after them gave 4 %. Measured, 32 / 8 heads, us: 2100 rows behind 7777 339 (790
// TFLOP/s), eight segments of 150 behind 1536 67, 146 rows behind 1536 26, 300 behind 100000 553. Against 64 bits, normal values, the
// first is 0.0023 off, where the result's rounding alone leaves 0.0016 and codes multiplied as they are (attn_decode4.hip) 0.0018: keys and
// values are rounded once more here.
//
// Fragment maps and ds_read_b64_tr_b16: attn_prefill.hip.

#include <algorithm>
#include <type_traits>

#include "kv4.h"

typedef _Float16 f16x8_mfma __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_mfma __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

#define QBLK 32
#define STAGE 128                  // keys staged per barrier round
#define NWAVES 8
#define STAGE_BYTES (STAGE * 256)  // K or V of a stage
#define CLASSES (4 * STAGE)        // bytes of a stage's: of K's and V's groups of each key
#define LDS_BYTES (4 * STAGE_BYTES + 2 * CLASSES + 2 * NWAVES)
#define PART_STRIDE 132            // of a row and head's partial: 128 sums, max, sum of exponentials
#define PART_ROWS (NWAVES * QBLK)  // rows and heads of an item and kv head

__device__ __forceinline__ int acc_row(int r, int half) { return (r & 3) + 8 * (r >> 2) + 4 * half; }   // C/D row map
// V's 32-byte slots of a row are XORed with this: the rows of a turned read, 4 by 2 slots, lie in all banks
__device__ __forceinline__ int v_turn(int row) { return (row & 3) * 2 + (row >> 2 & 1); }
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const f32x2 x = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2));
}
__device__ __forceinline__ f16x2 as_f16(uint32_t w) { return __builtin_bit_cast(f16x2, w); }

// An item of the plan: rows r0.. of a segment (first packed row, rows, its number), keys from..to of it, where its sums go (-1:
// nobody else has these rows)
struct Item {
  int row, len, r0, seg, from, to, part, unused;
};

// A group's class: the power of 2^16 that is taken out of it, after the largest exponent of its least value and step. A
// group of zeros or that is no number has none.
__device__ __forceinline__ int group_exponent(uint32_t w) {
  const int l = (int)(w >> 23 & 0xff), s = (int)(w >> 7 & 0xff);
  return l == 255 || s == 255 ? 0 : max(l, s ? s + 4 : 0);        // all values are below 2^(e - 127 + 2)
}
__device__ __forceinline__ bool has_no_class(int e) { return e == 0 || (e >= 117 && e <= 139); }
__device__ __forceinline__ int class_of_exponent(int e) {
  if (has_no_class(e)) return 0;
  e -= 127;
  return e > 12 ? (e - 13 >> 4) + 1 : max(-(-11 - e >> 4) - 1, -7);
}

// Four words of a row (32 values) to fp16, step and least value of each group: put(p, two words) takes those of nibble p, four
// neighbouring values
template <class P>
__device__ __forceinline__ void kv4_to_f16(const u32x4& w, const f32x2 (&scales)[2], P put) {
  f16x2 step[2], least[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    step[g] = as_f16(pack_f16(scales[g][0], scales[g][0]));
    least[g] = as_f16(pack_f16(scales[g][1], scales[g][1]));
  }
  const f16x2 base = as_f16(0x64006400u);
  uint32_t mask = 0x000f000fu, magic = 0x64006400u;
  asm volatile("" : "+s"(mask), "+v"(magic));          // one instruction for both: it takes no two literals
#pragma unroll
  for (int up = 0; up < 2; ++up) {         // lower halves of the words, nibbles 0 to 3, then the upper ones
    uint32_t m[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) m[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], up ? 0x07060302 : 0x05040100);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      u32x2 v;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const f16x2 n = as_f16((m[i] >> 4 * p & mask) | magic) - base;
        v[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(n, step[p >> 1], least[p >> 1]));
      }
      put(up * 4 + p, v);
    }
  }
}

template <int GQA>
__global__ void __launch_bounds__(64 * NWAVES) attn_prefill4_kernel(
    bf16_t* __restrict__ out,              // [T, H, 128] contiguous
    float* __restrict__ parts,             // [parts, KVH, PART_ROWS, PART_STRIDE]
    const bf16_t* __restrict__ q,          // [T, H, 128], row stride q_stride
    const char* __restrict__ k_cache, const char* __restrict__ v_cache,            // [NB, KVH, BS, 64] bytes
    const uint32_t* __restrict__ k_scale, const uint32_t* __restrict__ v_scale,    // [NB, KVH, BS, 2] words (step, least)
    const Item* __restrict__ items, const int* __restrict__ block_tables, const int* __restrict__ seg_pos, float scale,
    int64_t q_stride, int block_size, uint32_t block_inverse, int max_blocks) {
  const int g_kv = blockIdx.x, num_kv_heads = gridDim.x;
  const Item it = items[blockIdx.y];
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = g_kv * GQA + wave % GQA;
  const int qrow0 = it.r0 + wave / GQA * QBLK, rows_end = min(it.len, it.r0 + NWAVES / GQA * QBLK);
  const int pos0 = seg_pos[it.seg];                      // keys before the segment's first row
  const bool active = qrow0 < rows_end;
  const int my_pos = pos0 + qrow0 + col;
  const int64_t held = (int64_t)max_blocks * block_size;
  // keys of this item that the group's last row sees, and this wave's
  const int end_grp = (int)min((int64_t)min(it.to, pos0 + rows_end), held);
  const int end_me = active ? min(end_grp, pos0 + min(rows_end, qrow0 + QBLK)) : 0;

  extern __shared__ __attribute__((aligned(1024))) char smem[];          // [buffer][K | V], classes [buffer][key][K's groups, V's], [buffer][wave] has any
  signed char* const classes = (signed char*)smem + 4 * STAGE_BYTES;
  signed char* const has_class = classes + 2 * CLASSES;

  // ---- Q fragments (B-operand), the row's largest element to 2^14 -------------------------------
  union Frag { u32x4 u; f16x8_mfma m; };
  Frag q_frag[8];
  float c2;                                // scores to base-2 exponents
  {
    const int row = active ? min(qrow0 + col, it.len - 1) : it.r0;
    const short* qp = (const short*)q + (int64_t)(it.row + row) * q_stride + h * 128 + half * 8;
    bf16x8_vec raw[8];
    float most = 0.0f;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      raw[s] = *reinterpret_cast<const bf16x8_vec*>(qp + s * 16);
#pragma unroll
      for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(bf16_to_f32(raw[s][j])));
    }
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(most), __float_as_uint(most), false, false);
    most = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
    const int e = max((int)(__float_as_uint(most) >> 23) - 127, -90);
    // a negative scale goes into Q's signs: the max below is taken before scaling
    const float up = ldexpf(scale < 0.0f ? -1.0f : 1.0f, 14 - e);
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) q_frag[s].u[j] = pack_f16(bf16_to_f32(raw[s][2 * j]) * up, bf16_to_f32(raw[s][2 * j + 1]) * up);
    // above zero, so that a masked score stays -inf
    c2 = fmaxf(ldexpf(fabsf(scale) * 1.44269504088896340736f, e - 14), 1e-37f);
  }
  const float THR2 = 8.0f * 1.44269504088896340736f;

  // ---- staging: a thread has 32 values of K row tid / 4 and of V's ------------------------------
  const int st_row = tid >> 2, st_part = tid & 3;
  const int* bt = block_tables + (int64_t)it.seg * max_blocks;
  auto block_of = [&](int key) {           // key / block_size by its reciprocal, which is off by one at most
    const int n = (int)__umulhi((uint32_t)key, block_inverse), rest = key - n * block_size;
    return n - (rest < 0) + (rest >= block_size);
  };
  auto key_at = [&](int ks) { return min(ks + st_row, end_grp - 1); };
  u32x4 kr, vr;
  u32x2 ksc, vsc;
  int block = 0;
  auto ask = [&](int ks) { block = bt[block_of(key_at(ks))]; };
  auto load = [&](int ks) {
    const int key = key_at(ks);
    const int64_t row = ((int64_t)block * num_kv_heads + g_kv) * block_size + (key - block_of(key) * block_size);
    kr = *reinterpret_cast<const u32x4*>(k_cache + row * KV4_BYTES + st_part * 16);
    vr = *reinterpret_cast<const u32x4*>(v_cache + row * KV4_BYTES + st_part * 16);
    ksc = *reinterpret_cast<const u32x2*>(k_scale + row * KV4_GROUPS);
    vsc = *reinterpret_cast<const u32x2*>(v_scale + row * KV4_GROUPS);
  };
  auto stage = [&](int buf) {
    // each of a row's four threads looks at one of its groups
    const uint32_t mine = st_part & 2 ? (st_part & 1 ? vsc[1] : vsc[0]) : (st_part & 1 ? ksc[1] : ksc[0]);
    const int e = group_exponent(mine);
    const bool any = __any(!has_no_class(e));
    // a V row that is no number: its key is made none, so that the rows that see it are none and the others do not meet it
    if (kv4_least(vsc[0]) != kv4_least(vsc[0]) || kv4_least(vsc[1]) != kv4_least(vsc[1]) || kv4_step(vsc[0]) != kv4_step(vsc[0]) ||
        kv4_step(vsc[1]) != kv4_step(vsc[1])) {
      ksc = u32x2{0x7fc07fc0u, 0x7fc07fc0u};
      vsc = u32x2{0u, 0u};
    }
    f32x2 k_by[2], v_by[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      k_by[g] = f32x2{kv4_step(ksc[g]), kv4_least(ksc[g])};
      v_by[g] = f32x2{kv4_step(vsc[g]), kv4_least(vsc[g])};
    }
    if (any) {
      const int c = class_of_exponent(e);
      classes[buf * CLASSES + st_row * 4 + st_part] = (signed char)c;
      const float down = ldexpf(1.0f, -16 * c);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        k_by[g] *= __shfl(down, (lane & ~3) + g);
        v_by[g] *= __shfl(down, (lane & ~3) + 2 + g);
      }
    }
    char* const k_to = smem + buf * 2 * STAGE_BYTES + st_row * 256;
    char* const v_to = k_to + STAGE_BYTES;
    // nibble p of words 4 part..: values 32 (p & 3) + 16 (p >> 2) + 4 part..
    kv4_to_f16(kr, k_by, [&](int p, const u32x2& v) {
      const int unit = 4 * (p & 3) + 2 * (p >> 2) + (st_part >> 1);
      *reinterpret_cast<u32x2*>(k_to + ((unit ^ (st_row & 15)) << 4) + (st_part & 1) * 8) = v;
    });
    kv4_to_f16(vr, v_by, [&](int p, const u32x2& v) {
      *reinterpret_cast<u32x2*>(v_to + (((2 * (p & 3) + (p >> 2)) ^ v_turn(st_row)) << 5) + st_part * 8) = v;
    });
    if (lane == 0) has_class[buf * NWAVES + wave] = any;
  };

  typedef __attribute__((address_space(3))) char* lds_t;
  typedef __attribute__((address_space(3))) const f16x8_mfma* lds_frag;
  typedef __attribute__((address_space(3))) s16x4* lds_turn;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_t)smem);
  // where this lane reads K (row col, unit half: the others are an XOR) and V turned (row (lane & 15) / 4 of its half's eight, 4
  // elements of 16)
  uint32_t k_get = lds0 + col * 256 + ((half ^ (col & 15)) << 4);
  uint32_t v_get = lds0 + STAGE_BYTES + (half * 8 + ((lane & 15) >> 2)) * 256 + ((((lane & 15) >> 2) * 2 ^ (lane >> 4 & 1)) << 5) + (lane & 3) * 8;
  // All of the item, up to a stage that has a group of another class than 0 (false); ANY: with such groups too. (As branches of one loop
  // they had all sums copied twice a tile: one of 2100 rows behind 7777 431 us.)
  auto run = [&](auto any_class) {
  constexpr bool ANY = decltype(any_class)::value;
  f32x16 o_acc[4] = {};
  float m_run = -INFINITY, l_run = 0.0f;
  auto tile = [&](int ks, int kt, int buf) {
    const uint32_t at = buf * 2 * STAGE_BYTES + (kt - ks) * 256;
    asm volatile("" : "+v"(k_get), "+v"(v_get));       // not all their addresses for the whole loop
    const bool plain = !ANY || __builtin_amdgcn_readfirstlane(*reinterpret_cast<const int*>(has_class + buf * NWAVES + (kt - ks) / 16)) == 0;
    // of key 8 (r >> 2) + .. of a half, where the four waves' rows have any; else what another stage left
    int half_now = half;
    asm volatile("" : "+v"(half_now));
    auto class_of = [&](int sub, int r, int of) {
      const int key = kt - ks + sub * 32 + acc_row(r, half_now);
      return has_class[buf * NWAVES + (key >> 4)] ? (int)classes[buf * CLASSES + key * 4 + of] : 0;
    };
    // ---- QK^T: S[key][qrow], 32 keys each ----------------------------
    f32x16 s_acc[2] = {};
    const uint32_t k_at = k_get + at;
    auto multiply_k = [&](int s, int sub, f32x16& acc) {         // row col + 32 sub has the same XOR
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(lds_frag)(uintptr_t)((k_at ^ (s << 5)) + sub * 32 * 256), q_frag[s].m, acc, 0, 0, 0);
    };
    if (!plain) {                          // a group at a time, its powers put back
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          f32x16 acc = {};
#pragma unroll
          for (int s = 4 * g; s < 4 * g + 4; ++s) multiply_k(s, sub, acc);
#pragma unroll
          for (int r = 0; r < 16; ++r) s_acc[sub][r] += ldexpf(acc[r], 16 * class_of(sub, r, g));
        }
    } else {
#pragma unroll
      for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) multiply_k(s, sub, s_acc[sub]);
    }
    if (kt + 64 > pos0 + qrow0 || kt + 64 > end_grp) {
      // rows see keys up to their own position, which also ends the segment
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = kt + sub * 32 + acc_row(r, half);
          if (key > my_pos || key >= end_grp) s_acc[sub][r] = -INFINITY;
        }
    }

    // ---- online softmax (row = lane-local) --------------------------------
    float tmax = s_acc[0][0];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int r = 0; r < 16; ++r) tmax = fmaxf(tmax, s_acc[sub][r]);
    {
      auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(tmax), __float_as_uint(tmax), false, false);
      tmax = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * c2;
    }
    // the running max is renewed per row (lane) and only when it grows by more than THR2
    float alpha = 1.0f;
    if (!(tmax <= m_run + THR2)) {
      const float m_new = fmaxf(m_run, tmax);
      alpha = (m_run == -INFINITY) ? 0.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
    }
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o_acc[dt][r] *= alpha;
      l_run *= alpha;
    }
    // masked scores: fma(-inf, c2, -m) = -inf, whose exponential is 0
    const float m_use = m_run == -INFINITY ? 0.0f : m_run;
    uint32_t pw[2][8];
    auto expo = [&](auto far) {
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int pr = 0; pr < 8; ++pr) {
          f32x2 p;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = s_acc[sub][2 * pr + e];
            if constexpr (far) {
              x *= c2;
              asm volatile("" : "+v"(x));  // a product of its own
              x -= m_use;
            } else {
              x = __builtin_fmaf(x, c2, -m_use);
            }
            p[e] = __builtin_amdgcn_exp2f(x);
            l_run += p[e];
          }
          pw[sub][pr] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, f16x2));
        }
    };
    // of a max beyond 2^18 the fma would leave what the max itself was rounded by, which is no small number any more
    if (__builtin_amdgcn_ballot_w64(fabsf(m_use) > 262144.0f)) expo(std::true_type());
    else expo(std::false_type());

    // ---- PV: O^T += V^T x P, 16 keys at a time ------------------------------
    const uint32_t v_at = v_get + at;
    auto fragment = [&](const uint32_t* w) {
      Frag pf;
      auto r0 = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
      auto r1 = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
      pf.u = u32x4{r0[0], r1[0], r0[1], r1[1]};
      return pf;
    };
    auto values = [&](int key, int dt) {
      union { s16x4 t[2]; f16x8_mfma m; } vf;
#pragma unroll
      for (int rd = 0; rd < 2; ++rd)
        vf.t[rd] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_turn)(uintptr_t)((v_at ^ (dt << 6) ^ (rd << 5)) + (key + rd * 4) * 256));
      return vf.m;
    };
    if constexpr (ANY) if (!plain) {       // V with its powers put back, and P, as two bf16 parts each, which hold fp16's bits
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int kw = 0; kw < 2; ++kw) {
          uint32_t* const w = &pw[sub][4 * kw];
          uint32_t parts2[2][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const f16x2 h2 = as_f16(w[j]);
            f32x2 x = {(float)h2[0], (float)h2[1]};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              parts2[e][j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2_t));
              x[0] -= __uint_as_float(parts2[e][j] << 16);
              x[1] -= __uint_as_float(parts2[e][j] & 0xffff0000u);
            }
            w[j] = 0u;                     // for the products below
          }
          union Frag16 { u32x4 u; bf16x8_mfma m; f16x8_mfma h; };
          const Frag16 p1 = {fragment(parts2[0]).u}, p2 = {fragment(parts2[1]).u};
#pragma unroll
          for (int dt = 0; dt < 4; ++dt) {
            Frag16 v, v1, v2;
            v.h = values(sub * 32 + kw * 16, dt);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const f16x2 h2 = as_f16(v.u[j]);
              f32x2 x;
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int key = kt - ks + sub * 32 + kw * 16 + half_now * 8 + 2 * j + e;
                x[e] = ldexpf((float)h2[e], has_class[buf * NWAVES + (key >> 4)] ? 16 * classes[buf * CLASSES + key * 4 + 2 + (dt >> 1)] : 0);
              }
              v1.u[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2_t));
              x[0] -= __uint_as_float(v1.u[j] << 16);
              x[1] -= __uint_as_float(v1.u[j] & 0xffff0000u);
              v2.u[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2_t));
            }
            o_acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v2.m, p2.m, o_acc[dt], 0, 0, 0);
            o_acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v2.m, p1.m, o_acc[dt], 0, 0, 0);
            o_acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v1.m, p2.m, o_acc[dt], 0, 0, 0);
            o_acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v1.m, p1.m, o_acc[dt], 0, 0, 0);
          }
        }
    }
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int kw = 0; kw < 2; ++kw) {
        const Frag pf = fragment(&pw[sub][4 * kw]);
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) o_acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(values(sub * 32 + kw * 16, dt), pf.m, o_acc[dt], 0, 0, 0);
      }
    __builtin_amdgcn_s_setprio(0);
  };

  int buf = 0;
  if (it.from < end_grp) {
    ask(it.from);
    load(it.from);
    ask(it.from + STAGE);
    stage(0);
    if (it.from + STAGE < end_grp) {
      load(it.from + STAGE);
      ask(it.from + 2 * STAGE);
    }
  }
  for (int ks = it.from; ks < end_grp; ks += STAGE, buf ^= 1) {
    // this stage is there, and the last one's buffer, whose reads have come back, is free
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if constexpr (!ANY) {
      const u32x2 has = *reinterpret_cast<const u32x2*>(has_class + buf * NWAVES);
      if (__builtin_amdgcn_readfirstlane(has[0] | has[1])) {
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");      // all have read it
        return false;
      }
    }
    auto next = [&] {
      if (ks + STAGE < end_grp) {
        stage(buf ^ 1);
        if (ks + 2 * STAGE < end_grp) {
          load(ks + 2 * STAGE);
          ask(ks + 3 * STAGE);
        }
      }
    };
    if (wave < NWAVES / 2) next();
    const int end = min(ks + STAGE, end_me);
#pragma unroll 1
    for (int kt = ks; kt < end; kt += 64) tile(ks, kt, buf);
    if (wave >= NWAVES / 2) next();        // the other wave of a SIMD: one makes keys while the other multiplies
  }

  // ---- merge half-sums, then the result or a partial ----------------------
  {
    auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
    l_run = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
  if (it.part >= 0) {
    float* const to = parts + (((int64_t)it.part * num_kv_heads + g_kv) * PART_ROWS + wave * QBLK + col) * PART_STRIDE;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int g2 = 0; g2 < 4; ++g2)       // regs 4*g2..+3 = d consecutive
        *reinterpret_cast<f32x4*>(to + dt * 32 + 8 * g2 + 4 * half) =
            f32x4{o_acc[dt][4 * g2], o_acc[dt][4 * g2 + 1], o_acc[dt][4 * g2 + 2], o_acc[dt][4 * g2 + 3]};
    if (half == 0) *reinterpret_cast<f32x2*>(to + 128) = f32x2{m_run, l_run};
  } else if (active && qrow0 + col < rows_end) {
    const float inv_l = l_run == 0.0f ? 0.0f : 1.0f / l_run;
    bf16_t* op = out + ((int64_t)(it.row + qrow0 + col) * (num_kv_heads * GQA) + h) * 128;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int g2 = 0; g2 < 4; ++g2) {
        bf16x4_vec o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = f32_to_bf16(o_acc[dt][4 * g2 + j] * inv_l);
        *reinterpret_cast<bf16x4_vec*>((short*)op + dt * 32 + 8 * g2 + 4 * half) = o;
      }
  }
  return true;
  };
  if (!run(std::false_type())) run(std::true_type());
}

// A group whose keys were cut: first packed row, rows, first part, parts
struct Cut {
  int row, rows, part, parts;
};

// 32 lanes for a row of a head, four dims a lane
__global__ void __launch_bounds__(256) attn_prefill4_merge_kernel(bf16_t* __restrict__ out, const float* __restrict__ parts,
                                                                  const Cut* __restrict__ cuts, int gqa) {
  const Cut c = cuts[blockIdx.y];
  const int g_kv = blockIdx.x, num_kv_heads = gridDim.x;
  const int d = (threadIdx.x & 31) * 4;
  const int i = blockIdx.z * 8 + (threadIdx.x >> 5);
  if (i < c.rows * gqa) {
    const int row = i / gqa, head = i % gqa;
    // row 32 t + r of head e lies in wave t * gqa + e
    const float* at = parts + (((int64_t)c.part * num_kv_heads + g_kv) * PART_ROWS + ((row >> 5) * gqa + head) * QBLK + (row & 31)) * PART_STRIDE;
    const int64_t step = (int64_t)num_kv_heads * PART_ROWS * PART_STRIDE;
    float M = -INFINITY;
#pragma unroll 8
    for (int p = 0; p < c.parts; ++p) M = fmaxf(M, at[p * step + 128]);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float l = 0.0f;
#pragma unroll 4
    for (int p = 0; p < c.parts; ++p) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(at + p * step + d);
      const f32x2 ml = *reinterpret_cast<const f32x2*>(at + p * step + 128);
      // a part whose keys none of these rows sees has no max and sums of 0; one that is no number has a sum that is none
      const float w = ml[0] == -INFINITY ? (ml[1] == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(ml[0] - M);
      l += ml[1] * w;
      acc += v * w;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    bf16x4_vec o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = f32_to_bf16(acc[r] * inv);
    *reinterpret_cast<bf16x4_vec*>((short*)out + ((int64_t)(c.row + row) * (num_kv_heads * gqa) + g_kv * gqa + head) * 128 + d) = o;
  }
}

// floats of an item's partial for each kv head
extern "C" int64_t attn_prefill4_part() { return (int64_t)PART_ROWS * PART_STRIDE; }

#define MAX_ITEMS 65535    // of a launch: they lie on the grid's y

// items [n, 8] and cuts [m, 4] int32 on the device. 0, or -1 where the LDS cannot be had
extern "C" int launch_attn_prefill4(bf16_t* out, float* parts, const bf16_t* q, const void* k_cache, const void* v_cache,
                                    const void* k_scale, const void* v_scale, const int* items, int n, const int* cuts, int m,
                                    const int* block_tables, const int* seg_pos, float scale, int num_q_heads, int num_kv_heads,
                                    int64_t q_stride, int block_size, int max_blocks, hipStream_t stream) {
  const int gqa = num_q_heads / num_kv_heads;
  const uint32_t inverse = block_size > 1 ? (uint32_t)(((1ull << 32) + block_size - 1) / block_size) : ~0u;
  auto go = [&](auto kernel) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS_BYTES) != hipSuccess) return -1;
    for (int i = 0; i < n; i += MAX_ITEMS)
      hipLaunchKernelGGL(kernel, dim3(num_kv_heads, std::min(n - i, MAX_ITEMS)), dim3(64 * NWAVES), LDS_BYTES, stream, out, parts, q,
                         (const char*)k_cache, (const char*)v_cache, (const uint32_t*)k_scale, (const uint32_t*)v_scale,
                         reinterpret_cast<const Item*>(items) + i, block_tables, seg_pos, scale, q_stride, block_size, inverse, max_blocks);
    return 0;
  };
  if ((gqa == 1 ? go(attn_prefill4_kernel<1>) : gqa == 2 ? go(attn_prefill4_kernel<2>) : gqa == 4 ? go(attn_prefill4_kernel<4>)
                                                                                                  : go(attn_prefill4_kernel<8>)) != 0)
    return -1;
  for (int i = 0; i < m; i += MAX_ITEMS)
    hipLaunchKernelGGL(attn_prefill4_merge_kernel, dim3(num_kv_heads, std::min(m - i, MAX_ITEMS), PART_ROWS / 8), dim3(256), 0, stream, out, parts,
                       reinterpret_cast<const Cut*>(cuts) + i, gqa);
  return 0;
}
