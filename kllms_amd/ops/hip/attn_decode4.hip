// Paged decode attention (one query row for each stream) against a cache held in 4 bits (kv4.h), for gfx950.
//
// With k_td = n_td s_tg + m_tg for the values d of group g, n a whole number of 0..15:
//
//   score_t = sum_g s_tg (sum_d q_d n_td) + m_tg (sum_d q_d)      out_d = sum_t (p_t s_tg) n_td + sum_t p_t m_tg
//
// so the matrix cores multiply the whole numbers themselves, and step and least value meet sums, not elements: five
// vector instructions for the eight values of a word, where a value at a time takes two each and a product. A nibble masked out of its
// half of a word is an fp16 number as it stands, n * 2^-24 (below the normal ones, which the matrix cores take as they
// are), or 16 times that, which the other operand or the end makes good. q and p s are fp16 too: q's 8 bits are exact
// once its largest is scaled into fp16's range, p s is rounded to 11 bits, at most 2^-11 of each, an eighth of
// the result's own rounding. Measured against 64 bits, normal values: 0.0018 where that rounding alone leaves 0.0016.
//
// A wave takes 64 keys at a time and keeps its own running max and sum; four waves to a workgroup, Z workgroups to a context
// (deal, attn_decode4_slots), merged by the last of them to arrive or by a second launch where the caller has no counters.
//
//   scores   S[key][column] (16x16x32), column n is head n % GQA in set n / GQA. All sets hold the same scores; set j
//            works on GQA of a lane's 16 alone: no exponential is computed twice, a lane loads the scales of GQA keys
//   P V      O^T = V^T P^T: P's columns have the keys of their set and zeros for the others, sets are added up at the end
//   max      renewed only when a score passes it by more than 8 (in powers of two)
//   p s      is scaled to fp16's range by its own largest so far, of each head and group, renewed in the same way
//
// A wave's tile goes to a strip of LDS that is its own, straight from memory and as it lies there: nine loads of whole lines
// for 64 keys, without registers in between or barriers; the next K is on its way as soon as this one's fragments are read, the next V
// behind P V. (Loaded to registers by the fragments' own pattern, 4 + 16 + 16 loads whose lanes lie in many rows, the address
// unit was the bound: 16 streams of 6100 33 us, one of 131071 with eight heads to a kv head 48.) A row's 16-byte units are
// XORed with its key: both kinds of reads are free of bank conflicts. Key 4 r + c of 16 is row 4 c + r of a score tile.
//
// What bounds it: the cache's bytes where contexts are long, the vector units (58 % of their time, the waves waiting for
// 39 % of theirs) where they are many, else the chain of loads of one tile. Measured, us: one
// context of 150, 16 / 4 heads 6.3; 120 of 520 to 577 of which five each share 512, 32 / 8 heads 18.0 (83 MB from the L2s, 27 from behind
// them); 16 of 4500 to 7777 30.5 (120 MB, 4.5 TB/s, and a launch that joins shares); one of 131071, 64 / 8 heads 32.9 (151 MB, 5.2 TB/s, and that launch).

#include <algorithm>

#include "kv4.h"

typedef _Float16 f16x8_mfma __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_cvt __attribute__((ext_vector_type(2)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

#define NTHREADS 256
#define TKEYS 64           // keys of a wave's tile
#define PART_STRIDE 132    // of a head's partial: 128 sums, max, sum of exponentials
#define FAR 16             // loads and stores past the L2, from and to other XCDs' workgroups
#define LAG 8.0f           // how far a score may pass the running max, in powers of two
#define ROOM 32768.0f      // largest p s in fp16
#define SPARE 4            // powers of two that p s may grow by before it is scaled anew
// Bytes of a layer's keys and values from which on they are loaded with the streaming hint (nt), where no neighbour shares the
// prompt. us without and with: 16 streams of 6144, 32 / 8 heads 31.9, 27.7; one of 131072, 64 / 8 heads 46.2, 44.7
#define ONCE (16 << 20)
#define ROW_BYTES 144      // of a key and its value
#define LOG2E 1.44269504088896340736f

union Frag4 {
  u32x4 u;
  f16x8_mfma m;
};

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const f32x2 x = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2_cvt));
}

// Who works on what: a kv head's ``slots`` workgroups are dealt out, a context having one for every so many of its tiles, so that
// contexts of different lengths keep the chip equally busy. Of the three numbers of tiles that come of all slots, of half a slot less for
// each row and of one less, the least that keeps to the slots; the third one always does. Every wave counts for itself, by
// register moves, up to four rows a lane; more rows than that have one workgroup each. (With the same number for all contexts, and idle
// workgroups between those at work, compute units had one to three of them: 16 streams of 4500 to 7777 32.9 us, of 6144 28.0.)
#define DEAL_ROWS 256
struct Deal {
  int row, length, share, shares, start;   // workgroups of the row, from slot ``start`` on; row -1: nobody's slot
};
__device__ __forceinline__ int tiles_of(int length) { return (int)(((int64_t)length + TKEYS - 1) / TKEYS); }
// any number does, as long as all agree: the tiles go round. Joining shares takes 2 us, a round of four tiles 1.9: those that
// save less than two rounds are not made (one context of 530 8.9 us in three, 10.3 in one)
__device__ __forceinline__ int shares_of(int tiles, float inverse) {
  // written as the operations that they are: both kernels have to come to the same number
  const int n = max((int)ceilf(__builtin_fmaf((float)tiles, inverse, -1e-3f)), 1);
  const float rounds = ceilf(__builtin_fmaf(tiles * 0.25f, __builtin_amdgcn_rcpf((float)n), -1e-3f));
  return tiles > 8 && ceilf(tiles * 0.25f) - rounds >= 2.0f ? n : 1;
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ int lane_moved(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int scan(int x) {             // of this lane's and those before it
  x += lane_moved<0x111>(x);               // row_shr 1
  x += lane_moved<0x112>(x);               // 2
  x += lane_moved<0x114>(x);               // 4
  x += lane_moved<0x118>(x);               // 8
  x += lane_moved<0x142, 0xa>(x);          // row_bcast 15
  x += lane_moved<0x143, 0xc>(x);          // row_bcast 31
  return x;
}
__device__ __forceinline__ int last_lane(int x) { return __builtin_amdgcn_readlane(x, 63); }
// BY_ROW: of row ``at``; else of slot ``at``. EACH: rows of a lane
template <bool BY_ROW, int EACH>
__device__ __forceinline__ Deal deal_rows(const int* __restrict__ lengths, int B, int kv_heads, int64_t limit, int slots, int at) {
  const int lane = threadIdx.x & 63;
  int length[EACH], z[EACH], n = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int row = lane * EACH + e;
    length[e] = row < B ? (int)min((int64_t)max(lengths[row], 0), limit) : 0;
    n += tiles_of(length[e]);
  }
  // Not more workgroups than there are four tiles for; of many contexts, which fill the chip as they are, more tiles: a sixteenth of how
  // many there are, but of contexts that are longer than most as many as most have. 32 / 8 heads, us: 32 of 1000 15.9 in two shares each,
  // 13.8 in one; 16 of 1000 13.0 in four, 12.7 in two; 24 of 530 14.4 in two and three, 11.4 in one
  const float all = (float)max(last_lane(scan(n)), 1);
  const float most = __builtin_amdgcn_rcpf(fmaxf(4.0f, fminf((float)B * kv_heads * (1.0f / 16), all * 1.5f * __builtin_amdgcn_rcpf((float)B))));
  auto inverse = [&](float of) { return fminf(__builtin_amdgcn_rcpf(all) * of, most); };
  const float per0 = inverse(slots), per1 = inverse(slots - 0.5f * B);
  n = 0;                                   // slots by the first and by the second, 16 bits each
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if (lane * EACH + e < B)
      n += shares_of(tiles_of(length[e]), per0) + (shares_of(tiles_of(length[e]), per1) << 16);      // both below slots + B
  n = last_lane(scan(n));
  const float per = (n & 0xffff) <= slots ? per0 : n >> 16 <= slots ? per1 : inverse(slots - B);
  n = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    z[e] = lane * EACH + e < B ? shares_of(tiles_of(length[e]), per) : 0;
    n += z[e];
  }
  const int until = scan(n);               // slots of this lane's rows end here
  const int who = BY_ROW ? at / EACH : __popcll(__ballot(until <= at));
  Deal d = {-1, 0, 0, 1, 0};
  if (who >= 64) return d;
  int from = __builtin_amdgcn_readlane(until, who) - __builtin_amdgcn_readlane(n, who);
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int m = __builtin_amdgcn_readlane(z[e], who), l = __builtin_amdgcn_readlane(length[e], who);
    if (BY_ROW ? who * EACH + e == at : at >= from && at < from + m) d = Deal{who * EACH + e, l, at - from, m, from};
    from += m;
  }
  return d;
}
template <bool BY_ROW>
__device__ __forceinline__ Deal deal(const int* __restrict__ lengths, int B, int kv_heads, int64_t limit, int slots, int at) {
  if (slots <= B) return Deal{at, (int)min((int64_t)max(lengths[at], 0), limit), 0, 1, at};
  if (B == 1) {
    const int length = (int)min((int64_t)max(lengths[0], 0), limit), n = min(shares_of(tiles_of(length), 0.25f), slots);
    return Deal{BY_ROW || at < n ? 0 : -1, length, at, n, 0};
  }
  return B <= 64 ? deal_rows<BY_ROW, 1>(lengths, B, kv_heads, limit, slots, at)
                 : deal_rows<BY_ROW, DEAL_ROWS / 64>(lengths, B, kv_heads, limit, slots, at);
}

// The partials [GQA, PART_STRIDE] of Z workgroups, ``apart`` floats from each other, in their order, to rows of the result,
// by all threads. DEEP of them are asked for before the first is waited for, in fours that are there (all 16, there or not, and
// stores of 4 bytes before it: 1 us more)
template <int GQA, int DEEP>
__device__ __forceinline__ void merge4(bf16_t* __restrict__ out, const float* all, int Z, int apart, float (&sums)[NTHREADS][4],
                                       float (&ml)[NTHREADS][2]) {
  constexpr int SETS = NTHREADS / (32 * GQA);
  const int tid = threadIdx.x, h = (tid >> 5) % GQA, d = (tid & 31) * 4, set = tid / (32 * GQA);
  const auto far = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(all), 0, ((Z - 1) * apart + GQA * PART_STRIDE) * 4, 0x00020000);
  float M = -INFINITY, sum = 0.0f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int z0 = set; z0 < Z; z0 += DEEP * SETS) {
    f32x4 part[DEEP];
    f32x2 of[DEEP];
#pragma unroll
    for (int e0 = 0; e0 < DEEP; e0 += 4)
      if (z0 - set + e0 * SETS < Z) {      // the same for all threads
#pragma unroll
        for (int e = e0; e < e0 + 4; ++e) {  // behind the last one zeros
          const int at = ((z0 + e * SETS) * apart + h * PART_STRIDE) * 4;
          of[e] = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(far, at + 512, 0, FAR));
          part[e] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(far, at + d * 4, 0, FAR));
        }
      }
    const float before = M;
#pragma unroll
    for (int e = 0; e < DEEP; ++e)
      if (z0 + e * SETS < Z) M = fmaxf(M, of[e][0]);
    const float a = before == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(before - M);
    sum *= a;
    acc *= a;
#pragma unroll
    for (int e = 0; e < DEEP; ++e)
      if (z0 + e * SETS < Z) {
        const float w = of[e][0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(of[e][0] - M);
        sum += of[e][1] * w;
        acc += part[e] * w;
      }
  }
  if constexpr (SETS > 1) {
#pragma unroll
    for (int r = 0; r < 4; ++r) sums[tid][r] = acc[r];
    ml[tid][0] = M;
    ml[tid][1] = sum;
    __syncthreads();
    if (set > 0) return;
    float top = M;
#pragma unroll
    for (int e = 1; e < SETS; ++e) top = fmaxf(top, ml[tid + e * 32 * GQA][0]);
    const float a = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - top);
    sum *= a;
    acc *= a;
#pragma unroll
    for (int e = 1; e < SETS; ++e) {
      const float m = ml[tid + e * 32 * GQA][0], w = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
      sum += ml[tid + e * 32 * GQA][1] * w;
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] += sums[tid + e * 32 * GQA][r] * w;
    }
  }
  bf16x4_vec v;
  // no key at all: zeros. (A sum that is no number stays none)
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = f32_to_bf16(sum == 0.0f ? 0.0f : acc[r] / sum);
  *reinterpret_cast<bf16x4_vec*>((short*)out + h * 128 + d) = v;
}

// WHOLE: blocks of a multiple of 16 keys
template <int GQA, bool WHOLE>
__global__ __launch_bounds__(NTHREADS, GQA == 8 || !WHOLE ? 3 : 4) void attn_decode4_kernel(
    float* __restrict__ partials,          // [slots, KVH, GQA, PART_STRIDE]
    bf16_t* __restrict__ out,              // written where one workgroup has the context, or by the last one with ``arrived``
    const bf16_t* __restrict__ q,          // [B, H, 128], row stride q_stride
    const uint32_t* __restrict__ k_cache, const uint32_t* __restrict__ v_cache,    // [NB, KVH, BS, 16] words
    const uint32_t* __restrict__ k_scale, const uint32_t* __restrict__ v_scale,    // [NB, KVH, BS, 2] words (step, least)
    const int* __restrict__ block_tables, const int* __restrict__ context_lens, int* __restrict__ arrived, int apart,
    float scale, int block_size, uint32_t block_inverse, int max_blocks, int64_t q_stride, int B, int slots) {
  constexpr int SETS = 16 / GQA;
  constexpr int STRIP = 2 * TKEYS * KV4_BYTES + 2 * TKEYS * 8;
  static_assert(STRIP >= 16 * PART_STRIDE * 4);
  __shared__ __attribute__((aligned(1024))) char strips[4][STRIP];
  float (&o_lds)[4][STRIP / 4] = reinterpret_cast<float(&)[4][STRIP / 4]>(strips);      // at the end: a wave's sums, [16][PART_STRIDE]
  __shared__ float m_lds[4][16], l_lds[4][16];
  __shared__ int last_lds;
  const int g_kv = blockIdx.x, num_kv_heads = gridDim.x;
  const Deal mine = deal<false>(context_lens, B, num_kv_heads, (int64_t)max_blocks * block_size, slots, blockIdx.y);
  const int b = __builtin_amdgcn_readfirstlane(mine.row), z = __builtin_amdgcn_readfirstlane(mine.share);
  const int Z = __builtin_amdgcn_readfirstlane(mine.shares), L = __builtin_amdgcn_readfirstlane(mine.length);
  if (b < 0) return;
  const int tiles = tiles_of(L);
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head = col % GQA, set = col / GQA;

  // ---- q: largest element to 2^14, exponents that fp16 holds; sums of its groups -------------
  Frag4 qf[4];
  float q_back, q_sum[2];
  {
    const short* qp = (const short*)q + (int64_t)b * q_stride + (g_kv * GQA + head) * 128 + grp * 4;
    bf16x4_vec raw[4][2];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int h = 0; h < 2; ++h) raw[a][h] = *reinterpret_cast<const bf16x4_vec*>(qp + a * 32 + h * 16);
    float most = 0.0f, sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = bf16_to_f32(raw[a][h][i]);
          most = fmaxf(most, fabsf(x));
          sum[a >> 1] += x;
        }
#pragma unroll
    for (int off = 16; off <= 32; off <<= 1) {
      most = fmaxf(most, __shfl_xor(most, off));
      sum[0] += __shfl_xor(sum[0], off);
      sum[1] += __shfl_xor(sum[1], off);
    }
    const int e = max((int)(__float_as_uint(most) >> 23) - 127, -90);
    const float up = ldexpf(1.0f, 14 - e);
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const float u = a & 1 ? up * 0.0625f : up;       // nibbles 1 and 3 of a half stand 16 times too high
#pragma unroll
      for (int i = 0; i < 4; ++i) qf[a].u[i] = pack_f16(bf16_to_f32(raw[a][0][i]) * u, bf16_to_f32(raw[a][1][i]) * u);
    }
    const float by = scale * LOG2E;
    q_back = ldexpf(by, e - 14 + 24);
    q_sum[0] = sum[0] * by;
    q_sum[1] = sum[1] * by;
  }

  // ---- which of a tile's keys this lane weighs: score tile tt_of(i), register r_of(i) ----------
  // GQA 8: r 2 set + (i & 1), tt i / 2; 4: r set, tt i; 2: r set & 3, tt 2 (set / 4) + i; 1: r set & 3, tt set / 4
  auto key_in_tile = [&](int i) {
    const int r = GQA == 8 ? 2 * set + (i & 1) : set & 3;
    const int tt = GQA == 8 ? i >> 1 : GQA == 4 ? i : GQA == 2 ? 2 * (set >> 2) + i : set >> 2;
    return 16 * tt + 4 * r + grp;
  };
  // where p goes in P's fragment: words 0 and 1 of a score tile's two, by register
  const int r_mine = GQA == 8 ? 2 * set : set & 3;
  const uint32_t half = GQA == 8 ? 0xffffffffu : r_mine & 1 ? 0xffff0000u : 0x0000ffffu;
  const uint32_t keep[2] = {r_mine < 2 ? half : 0u, r_mine < 2 ? 0u : half};

  const int* bt = block_tables + (int64_t)b * max_blocks;
  // the neighbours' first blocks are this context's: so are more, and lie in the L2
  const bool once = (int64_t)L * B * num_kv_heads * ROW_BYTES >= ONCE &&
                    !((b > 0 && bt[-max_blocks] == bt[0]) || (b + 1 < B && bt[max_blocks] == bt[0]));
  auto block_of = [&](int key) {           // key / block_size by its reciprocal, which is off by one at most
    const int n = (int)__umulhi((uint32_t)key, block_inverse), rest = key - n * block_size;
    return n - (rest < 0) + (rest >= block_size);
  };

  // ---- the strip: K of a tile, V, (step, least) of both -----------------------------------------
  char* const strip = strips[wave];
  typedef __attribute__((address_space(3))) char* lds_t;
  typedef __attribute__((address_space(3))) const u32x4* lds_v4;
  typedef __attribute__((address_space(3))) const u32x2* lds_v2;
  typedef __attribute__((address_space(3))) const uint32_t* lds_v1;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_t)strip);
  constexpr int V_AT = TKEYS * KV4_BYTES, S_AT = 2 * V_AT, VS_AT = S_AT + TKEYS * 8;
  // a load's lane has 16 bytes of row lane / 4 of sixteen
  const int put_row = lane >> 2;
  const uint32_t put_off = put_row * KV4_BYTES + (((lane & 3) ^ (put_row >> 2)) << 4);
  const int k_key = 4 * (col & 3) + (col >> 2);        // key of row ``col`` of a score tile
  uint32_t k_get = lds0 + k_key * KV4_BYTES + ((grp ^ (k_key >> 2)) << 4);
  uint32_t v_get = lds0 + V_AT + grp * KV4_BYTES + col * 4;          // word col of key grp, the unit XORed with the key's r
  uint32_t s_get = lds0 + S_AT + key_in_tile(0) * 8;
  auto put = [&](const char* rows, uint32_t lane_off, uint32_t at) {
    const uint64_t r = (uint64_t)rows;
    const u32x2 from = {(uint32_t)__builtin_amdgcn_readfirstlane((int)r), (uint32_t)__builtin_amdgcn_readfirstlane((int)(r >> 32))};
    if (once)
      asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(lane_off), "s"(from), "s"(at) : "memory");
    else
      asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(lane_off), "s"(from), "s"(at) : "memory");
  };
  auto put_at = [&](const char* from, uint32_t at) {
    if (once) asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(from), "s"(at) : "memory");
    else asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(at) : "memory");
  };
  auto put_word = [&](const uint32_t* from, uint32_t at) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(at) : "memory");
  };
  constexpr int IDS = WHOLE ? 4 : 1;
  int ids[IDS];                            // WHOLE: blocks of a tile's four sixteens; else the block of this lane's key
  auto ask = [&](int t) {
#pragma unroll
    for (int i = 0; i < IDS; ++i) {
      const int key = min(t * TKEYS + (WHOLE ? i * 16 : lane), L - 1);
      ids[i] = bt[block_of(key)];
    }
  };
  auto load_rows = [&](const uint32_t* cache, uint32_t to, const i32x4& base, int row) {    // 4 loads
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      if constexpr (WHOLE) {
        put((const char*)cache + (int64_t)base[tt] * KV4_BYTES, put_off, to + tt * 16 * KV4_BYTES);
      } else {
        const int64_t r = __shfl(row, 16 * tt + put_row);
        put_at((const char*)cache + r * KV4_BYTES + (((lane & 3) ^ (put_row >> 2)) << 4), to + tt * 16 * KV4_BYTES);
      }
    }
  };
  constexpr int SCALE_LOADS = WHOLE ? 1 : 4;
  auto load_scales = [&](const i32x4& base, int row) {
    if constexpr (WHOLE) {                 // two keys a lane, K's in the lower half of the wave
      const int at = lane & 31, tt = at >> 3;
      int r = base[0];
#pragma unroll
      for (int e = 1; e < 4; ++e) r = tt == e ? base[e] : r;
      put_at((const char*)(lane < 32 ? k_scale : v_scale) + ((int64_t)r * 8 + (at & 7) * 16), lds0 + S_AT);
    } else {                               // a word a lane
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t r = __shfl(row, (e & 1) * 32 + (lane >> 1));
        put_word((e < 2 ? k_scale : v_scale) + r * KV4_GROUPS + (lane & 1), lds0 + S_AT + e * 256);
      }
    }
  };
  // rows of the cache: of the four sixteens' first keys, or of this lane's key; those behind the context repeat what is in it
  auto rows_of = [&](int t, i32x4& base, int& row) {
    if constexpr (WHOLE) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = min(t * TKEYS + i * 16, (L - 1) & ~15);
        base[i] = __builtin_amdgcn_readfirstlane((ids[i] * num_kv_heads + g_kv) * block_size + (key - block_of(key) * block_size));
      }
    } else {
      const int key = min(t * TKEYS + lane, L - 1);
      row = (ids[0] * num_kv_heads + g_kv) * block_size + (key - block_of(key) * block_size);
    }
  };

  f32x4 o[8];
#pragma unroll
  for (int p = 0; p < 8; ++p) o[p] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.0f, low_run[2] = {0.0f, 0.0f};      // of this lane's head and keys
  float cap[2] = {0.0f, 0.0f}, to_cap[2] = {0.0f, 0.0f};       // what p s of a group stays below, and what it is multiplied by

  const int step = Z * 4;
  int t = z * 4 + wave;
  i32x4 base = {0, 0, 0, 0};
  int row = 0;
  if (t < tiles) {
    ask(t);
    rows_of(t, base, row);
    load_rows(k_cache, lds0, base, row);
    load_scales(base, row);
    load_rows(v_cache, lds0 + V_AT, base, row);
    ask(min(t + step, tiles - 1));
  }
#pragma unroll 1
  for (; t < tiles; t += step) {
    const bool more = t + step < tiles;
    if (more) {
      rows_of(t + step, base, row);
      ask(min(t + 2 * step, tiles - 1));
    }
    // ---- K's fragments and the scales are there (V is not): to registers, and the next ones on their way -------
    u32x4 kraw[4];
    u32x2 ks[GQA], vs[GQA];
    asm volatile("s_waitcnt vmcnt(4)" : "+v"(k_get), "+v"(v_get), "+v"(s_get)::"memory");      // not all their addresses for the whole loop
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) kraw[tt] = *(lds_v4)(uintptr_t)(k_get + tt * 16 * KV4_BYTES);
#pragma unroll
    for (int i = 0; i < GQA; ++i) {
      const int more_keys = GQA == 8 ? 16 * (i >> 1) + 4 * (i & 1) : 16 * i;     // key_in_tile(i) - key_in_tile(0)
      ks[i] = *(lds_v2)(uintptr_t)(s_get + more_keys * 8);
      vs[i] = *(lds_v2)(uintptr_t)(s_get + (VS_AT - S_AT) + more_keys * 8);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (more) {
      load_rows(k_cache, lds0, base, row);
      load_scales(base, row);
    }
    __builtin_amdgcn_sched_barrier(0);
    // ---- scores of whole numbers, a group at a time ---------------------------------------
    float x[GQA];
    {
      float sums[2][GQA];                  // of this lane's keys: of the registers of all sets, this one's
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        Frag4 f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = kraw[tt][i], w8 = w >> 8;
          f[0].u[i] = w & 0x000f000fu;
          f[1].u[i] = w & 0x00f000f0u;
          f[2].u[i] = w8 & 0x000f000fu;
          f[3].u[i] = w8 & 0x00f000f0u;
        }
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          f32x4 acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[2 * g].m, qf[2 * g].m, zero, 0, 0, 0);
          acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[2 * g + 1].m, qf[2 * g + 1].m, acc, 0, 0, 0);
          if constexpr (GQA == 8) {
            sums[g][2 * tt] = set ? acc[2] : acc[0];
            sums[g][2 * tt + 1] = set ? acc[3] : acc[1];
          } else {
            const float lo = set & 1 ? acc[1] : acc[0], hi = set & 1 ? acc[3] : acc[2], mine = set & 2 ? hi : lo;
            const int i = GQA == 4 ? tt : GQA == 2 ? tt & 1 : 0;
            if (GQA == 4 || tt < GQA) sums[g][i] = mine;
            else sums[g][i] = (GQA == 2 ? set >> 2 == tt >> 1 : set >> 2 == tt) ? mine : sums[g][i];
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < GQA; ++i) {
        const float whole = __builtin_fmaf(kv4_step(ks[i][1]), sums[1][i], kv4_step(ks[i][0]) * sums[0][i]);
        const float low = __builtin_fmaf(kv4_least(ks[i][1]), q_sum[1], kv4_least(ks[i][0]) * q_sum[0]);
        x[i] = __builtin_fmaf(whole, q_back, low);
      }
    }
    if (t * TKEYS + TKEYS > L) {           // what lies behind the context is another's
#pragma unroll
      for (int i = 0; i < GQA; ++i)
        if (t * TKEYS + key_in_tile(i) >= L) {
          x[i] = -INFINITY;
          vs[i] = u32x2{0u, 0u};
        }
    }
    // ---- the max, renewed when it has to be ----------------------------------------------------
    float top = x[0];
#pragma unroll
    for (int i = 1; i < GQA; ++i) top = fmaxf(top, x[i]);
    if (__any(top > m_run + LAG)) {
#pragma unroll
      for (int off = GQA; off <= 32; off <<= 1) top = fmaxf(top, __shfl_xor(top, off));
      const float m_new = fmaxf(m_run, top);
      const float alpha = m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        low_run[g] *= alpha;
        cap[g] *= alpha;                   // the sums stay as they are, in a smaller unit
        cap[g] = cap[g] < 1e-30f ? 0.0f : cap[g];
        to_cap[g] = cap[g] > 0.0f ? ROOM / cap[g] : 0.0f;
      }
    }
    // ---- P, and P times V's steps to fragments ------------------------------------------------
    const float m_use = m_run == -INFINITY ? 0.0f : m_run;
    Frag4 pf[2][2];                        // [32 keys][group]
    {
      float ps[GQA][2], wide[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < GQA; ++i) {
        const float p = __builtin_amdgcn_exp2f(x[i] - m_use);
        l_run += p;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          ps[i][g] = p * kv4_step(vs[i][g]);
          wide[g] = fmaxf(wide[g], ps[i][g]);
          low_run[g] = __builtin_fmaf(p, kv4_least(vs[i][g]), low_run[g]);
        }
      }
      if (__any(wide[0] > cap[0] || wide[1] > cap[1])) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
#pragma unroll
          for (int off = GQA; off <= 32; off <<= 1) wide[g] = fmaxf(wide[g], __shfl_xor(wide[g], off));
          float shrink = 1.0f;
          if (wide[g] > cap[g]) {
            const int e = min(max((int)(__float_as_uint(wide[g]) >> 23) - 126 + SPARE, -100), 127);
            const float cap_new = ldexpf(1.0f, e);
            shrink = cap[g] / cap_new;
            cap[g] = cap_new;
            to_cap[g] = ROOM / cap_new;
          }
#pragma unroll
          for (int p = 0; p < 8; ++p)
            if ((p & 3) >> 1 == g) o[p] *= shrink;
        }
      }
#pragma unroll
      for (int i = 0; i < GQA; ++i)
#pragma unroll
        for (int g = 0; g < 2; ++g) ps[i][g] *= to_cap[g];
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          uint32_t v;
          if constexpr (GQA == 8) {
            v = pack_f16(ps[2 * tt][g], ps[2 * tt + 1][g]);
          } else {
            const float one = ps[GQA == 4 ? tt : GQA == 2 ? tt & 1 : 0][g];
            v = pack_f16(one, one);
            if constexpr (GQA == 2) v = set >> 2 == tt >> 1 ? v : 0u;
            if constexpr (GQA == 1) v = set >> 2 == tt ? v : 0u;
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) pf[tt >> 1][g].u[(tt & 1) * 2 + e] = v & keep[e];
        }
    }
    // ---- P V: 32 keys at a time, a nibble a column tile, those of a word's lower half first -------
    if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(4 + SCALE_LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      uint32_t vraw[2][4];                 // word col of key 4 r + grp
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          vraw[tt][r] = *(lds_v1)(uintptr_t)((v_get ^ (r << 4)) + ((2 * s + tt) * 16 + 4 * r) * KV4_BYTES);
#pragma unroll
      for (int up = 0; up < 2; ++up) {
        __builtin_amdgcn_sched_barrier(0);
        Frag4 f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t a = vraw[e >> 1][(e & 1) * 2], c = vraw[e >> 1][(e & 1) * 2 + 1];
          const uint32_t w = __builtin_amdgcn_perm(c, a, up ? 0x07060302 : 0x05040100), w8 = w >> 8;
          f[0].u[e] = w & 0x000f000fu;
          f[1].u[e] = w & 0x00f000f0u;
          f[2].u[e] = w8 & 0x000f000fu;
          f[3].u[e] = w8 & 0x00f000f0u;
        }
#pragma unroll
        for (int p = 0; p < 4; ++p)
          o[up * 4 + p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[p].m, pf[s][p >> 1].m, o[up * 4 + p], 0, 0, 0);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (more) load_rows(v_cache, lds0 + V_AT, base, row);
    __builtin_amdgcn_sched_barrier(0);
  }

  // ---- this wave's sums, then the sets' and the waves' ------------------------------------------
#pragma unroll
  for (int off = 16; off <= 32; off <<= 1) {
    l_run += __shfl_xor(l_run, off);
    low_run[0] += __shfl_xor(low_run[0], off);
    low_run[1] += __shfl_xor(low_run[1], off);
  }
  const float back[2] = {cap[0] * (16777216.0f / ROOM), cap[1] * (16777216.0f / ROOM)};       // 2^24: the nibbles'
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const int g = (p & 3) >> 1;
    f32x4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = __builtin_fmaf(o[p][r], p & 1 ? back[g] * 0.0625f : back[g], low_run[g]);
    *reinterpret_cast<f32x4*>(&o_lds[wave][col * PART_STRIDE + 32 * (p & 3) + 16 * (p >> 2) + 4 * grp]) = v;
  }
  if (lane < 16) {
    m_lds[wave][lane] = m_run;
    l_lds[wave][lane] = l_run;
  }
  __syncthreads();
  float* const part = partials + ((int64_t)blockIdx.y * num_kv_heads + g_kv) * (GQA * PART_STRIDE);
  bf16_t* const to = out + ((int64_t)b * num_kv_heads + g_kv) * GQA * 128;
  constexpr int VEC = GQA > 2 ? GQA / 2 : 1;
  if (tid * VEC < GQA * 128) {
    const int h = tid * VEC >> 7, d = tid * VEC & 127;
    float M = m_lds[0][h];
#pragma unroll
    for (int w = 1; w < 4; ++w) M = fmaxf(M, m_lds[w][h]);
    float acc[VEC] = {}, l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float e = m_lds[w][h] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_lds[w][h] - M);
#pragma unroll
      for (int j = 0; j < SETS; ++j) {
        l += l_lds[w][h + GQA * j] * e;
#pragma unroll
        for (int r = 0; r < VEC; ++r) acc[r] += o_lds[w][(h + GQA * j) * PART_STRIDE + d + r] * e;
      }
    }
    if (Z == 1) {
#pragma unroll
      for (int r = 0; r < VEC; ++r) ((short*)to)[h * 128 + d + r] = f32_to_bf16(l == 0.0f ? 0.0f : acc[r] / l);
    } else {
      const auto far = __builtin_amdgcn_make_buffer_rsrc(part, 0, GQA * PART_STRIDE * 4, 0x00020000);
      const int at = (h * PART_STRIDE + d) * 4;
      if constexpr (VEC == 4)
        __builtin_amdgcn_raw_buffer_store_b128(u32x4{__float_as_uint(acc[0]), __float_as_uint(acc[1]), __float_as_uint(acc[2]), __float_as_uint(acc[3])},
                                              far, at, 0, FAR);
      else if constexpr (VEC == 2)
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(acc[0]), __float_as_uint(acc[1])}, far, at, 0, FAR);
      else
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(acc[0]), far, at, 0, FAR);
      if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(u32x2{__float_as_uint(M), __float_as_uint(l)}, far, (h * PART_STRIDE + 128) * 4, 0, FAR);
    }
  }
  if (Z == 1 || !arrived) return;
  // ---- the last workgroup to arrive merges the partials ------------------------------------------
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    int* const count = arrived + ((int64_t)b * num_kv_heads + g_kv) * apart;
    last_lds = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == Z - 1;
    if (last_lds) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last_lds) return;
  merge4<GQA, 8>(to, part - (int64_t)z * num_kv_heads * (GQA * PART_STRIDE), Z, num_kv_heads * (GQA * PART_STRIDE),
              reinterpret_cast<float(&)[NTHREADS][4]>(o_lds[0]), reinterpret_cast<float(&)[NTHREADS][2]>(o_lds[1]));
}

// the same in a launch of its own, a workgroup for each head
__global__ __launch_bounds__(NTHREADS) void attn_decode4_merge_kernel(bf16_t* __restrict__ out, const float* __restrict__ partials,
                                                                     const int* __restrict__ context_lens, int64_t limit, int B,
                                                                     int kv_heads, int slots) {
  __shared__ float sums[NTHREADS][4], ml[NTHREADS][2];
  const int h = blockIdx.x, num_q_heads = gridDim.x, b = blockIdx.y;
  const Deal mine = deal<true>(context_lens, B, kv_heads, limit, slots, b);
  const int Z = __builtin_amdgcn_readfirstlane(mine.shares);
  if (Z == 1) return;                      // its one workgroup has written the result
  merge4<1, 16>(out + ((int64_t)b * num_q_heads + h) * 128,
            partials + ((int64_t)__builtin_amdgcn_readfirstlane(mine.start) * num_q_heads + h) * PART_STRIDE, Z, num_q_heads * PART_STRIDE,
            sums, ml);
}

// rows of a launch: they lie on the grid's y, which ends at 65535
#define MAX_ROWS 65535

// Workgroups of a kv head: two for each compute unit, a workgroup's beginning and end being 5 us of its own; of more rows than
// units one for each, and some for contexts that are much longer than the others. us in all of 256, 512, 768 and 1024 workgroups: 16
// streams of 6144, 32 / 8 heads 27.1, 25.6, 27.8, 27.7; one of 131072, 64 / 8 heads 40.9, 33.9, 38.9, 38.1; 40 of 1500 (320 pairs) 18.5 with
// a workgroup each, 22.2 with two. max_ctx: positions of the table
static int attn_decode4_slots(int B, int num_kv_heads, int64_t max_ctx) {
  const int slots = std::max(1, 512 / num_kv_heads);
  // contexts of a few rounds at most are as they are where they fill the chip
  if (B > DEAL_ROWS || max_ctx <= 4 * TKEYS || (2 * B > slots && max_ctx <= 16 * TKEYS)) return B;
  if (B == 1) return (int)std::min<int64_t>(slots, (max_ctx + 4 * TKEYS - 1) / (4 * TKEYS));
  return 2 * B <= slots ? slots : B + std::max(1, 256 / num_kv_heads);
}

// floats of a launch's partials: 0 where every row has one workgroup
extern "C" int64_t attn_decode4_room(int B, int num_kv_heads, int gqa, int64_t max_ctx) {
  const int slots = attn_decode4_slots(B, num_kv_heads, max_ctx);
  return slots > B ? (int64_t)slots * num_kv_heads * gqa * PART_STRIDE : 0;
}

extern "C" void launch_attn_decode4(bf16_t* out, float* partials, int* arrived, int apart, const bf16_t* q, const void* k_cache,
                                    const void* v_cache, const void* k_scale, const void* v_scale, const int* block_tables,
                                    const int* context_lens, float scale, int num_q_heads, int num_kv_heads, int block_size,
                                    int max_blocks, int64_t q_stride, int B, hipStream_t stream) {
  const int gqa = num_q_heads / num_kv_heads;
  const int64_t limit = (int64_t)max_blocks * block_size;
  // more than B of at most DEAL_ROWS rows, which are one launch; else every row of a launch has one workgroup, whatever the others'
  const int dealt = attn_decode4_slots(B, num_kv_heads, limit);
  // merged by the last workgroup, unless its work alone is more than a launch: heads times shares of a context
  if ((int64_t)(dealt / B) * gqa > 192) arrived = nullptr;
  const uint32_t inverse = block_size > 1 ? (uint32_t)(((1ull << 32) + block_size - 1) / block_size) : ~0u;
  for (int b0 = 0; b0 < B; b0 += MAX_ROWS) {
    const int rows = B - b0 < MAX_ROWS ? B - b0 : MAX_ROWS, slots = dealt > B ? dealt : rows;
    const dim3 grid(num_kv_heads, slots);
    bf16_t* o = out + (int64_t)b0 * num_q_heads * 128;
    const bf16_t* q0 = q + (int64_t)b0 * q_stride;
    const int* bt = block_tables + (int64_t)b0 * max_blocks;
#define LAUNCH(G, W)                                                                                                    \
  hipLaunchKernelGGL((attn_decode4_kernel<G, W>), grid, dim3(NTHREADS), 0, stream, partials, o, q0, (const uint32_t*)k_cache, \
                     (const uint32_t*)v_cache, (const uint32_t*)k_scale, (const uint32_t*)v_scale, bt, context_lens + b0, arrived,  \
                     apart, scale, block_size, inverse, max_blocks, q_stride, rows, slots)
#define DISPATCH(G)                                                                                                       \
  do {                                                                                                                    \
    if (block_size % 16 == 0) LAUNCH(G, true);                                                                            \
    else LAUNCH(G, false);                                                                                                \
  } while (0)
    switch (gqa) {
      case 1: DISPATCH(1); break;
      case 2: DISPATCH(2); break;
      case 4: DISPATCH(4); break;
      default: DISPATCH(8); break;
    }
#undef DISPATCH
#undef LAUNCH
    if (slots > rows && !arrived)
      hipLaunchKernelGGL(attn_decode4_merge_kernel, dim3(num_q_heads, rows), dim3(NTHREADS), 0, stream, o, partials, context_lens + b0, limit,
                         rows, num_kv_heads, slots);
  }
}
