// Products of rows in 8-bit integers, a scale for each row, with a weight matrix in 8-bit integers, a scale for each of its
// rows (output channels), for gfx950:
//
//   s_m = max |x_m| / 127,  c_m = x_m / s_m to the nearest whole number, halves to even
//   y_mn = (sum_k c_mk w_nk) s_m t_n (+ b_n),  or silu(gate) * up of such sums in fp32, rounded once
//
// The sums are of 32 bits and exact: 127 * 127 * K stays below 2^31 up to K = 131072. So shares of K add up to the same
// whoever is last. 127 x and its quotient by max |x| decide between two whole numbers as the exact quotient does: both are bf16
// values, of 8 bits, so a quotient that is no half itself is 2^-17 of it away from one.
//
// On the ring and tiles of tile_product.h, to which a row of K integers is one of K / 2 bf16: as many bytes and
// matrix instructions of twice the products. Where W's stream or the depth of K is the bound, tiles of 64 or 128 rows of W
// (linear_rows.hip has the reasons), two workgroups to a compute unit where the ring leaves room; else tiles of 256 and the
// matrix units (linear_tiles.hip). int8_plan weighs them. Up to 8 rows go in one launch that makes the codes too (int8_few). A
// product of few tiles is shared out over K: each workgroup leaves its sums past the L2 and the last one to arrive adds them up.
// The counters for that are zeroed by the launch that makes the codes, which comes before anyway.
//
// Measured, us: 6144 x 4096, 5 rows 7.9 (25 MB, 3.2 TB/s); 28672 x 4096 with the activation, 120 rows 34 (W at 3.9 TB/s), 7777 rows 790
// (2310 TOP/s, the card's power limit; the library's 8192^3 has 2083); 4608 x 3584 with bias, 333 rows 17.8.
//
// K is a multiple of 16; the codes' rows are filled up to whole stages with zeros, which what W has behind a row meets.

#include <atomic>

#include "int8.h"
#include "tile_product.h"


#define LI_STAGE 128       // bytes of a row in a stage
enum Int8Form { LI_BF16 = 0, LI_SILU = 1, LI_PART = 2 };

// ---- codes ---------------------------------------------------------------------------------------

// LANES threads a row, R vectors of 8 of each (R 0: any number, read twice). codes [M, padded], zeros behind K; clears
// ``clear`` beside.
template <int LANES, int R>
__global__ void __launch_bounds__(256) int8_rows_kernel(int8_t* __restrict__ codes, float* __restrict__ scales,
                                                        const bf16_t* __restrict__ x, int64_t x_stride, int M, int K, int padded,
                                                        int* __restrict__ clear, int clears) {
  __shared__ uint32_t red[4];
  const int tid = threadIdx.x, lane = tid % LANES;
  for (int i = blockIdx.x * 256 + tid; i < clears; i += gridDim.x * 256) clear[i] = 0;
  const int m = blockIdx.x * (256 / LANES) + tid / LANES;
  if (LANES == 64 && m >= M) return;
  const int vecs = K / 8, all = padded / 8;
  const u16x8* row = reinterpret_cast<const u16x8*>((const short*)x + (int64_t)m * x_stride);
  u32x2* to = reinterpret_cast<u32x2*>(codes + (int64_t)m * padded);
  u16x8 v[R > 0 ? R : 1];
  u16x8 top = {};
  if constexpr (R > 0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = lane + r * LANES;
      v[r] = i < vecs ? row[i] : u16x8{};
    }
#pragma unroll
    for (int r = 0; r < R; ++r) top = __builtin_elementwise_max(top, v[r] & (u16x8)(unsigned short)0x7fff);
  } else {
    for (int i = lane; i < vecs; i += LANES) top = __builtin_elementwise_max(top, row[i] & (u16x8)(unsigned short)0x7fff);
  }
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) most = max(most, (uint32_t)top[j]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, off));
  if constexpr (LANES == 256) {
    if ((tid & 63) == 0) red[tid >> 6] = most;
    __syncthreads();
    most = max(max(red[0], red[1]), max(red[2], red[3]));
  }
  const Int8Row by(most);
  if (lane == 0) scales[m] = by.scale;
  auto put = [&](int i, const u16x8& a) { to[i] = by.codes(a); };
  if constexpr (R > 0) {
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (lane + r * LANES < all) put(lane + r * LANES, v[r]);
  } else {
    for (int i = lane; i < all; i += LANES) put(i, i < vecs ? row[i] : u16x8{});
  }
}

extern "C" int int8_rows_padded(int K) { return (K + LI_STAGE - 1) / LI_STAGE * LI_STAGE; }

extern "C" void launch_int8_rows(int8_t* codes, float* scales, const bf16_t* x, int64_t x_stride, int M, int K, int* clear, int clears,
                                 hipStream_t stream) {
  const int padded = int8_rows_padded(K);
#define LI_ROWS(LANES, R)                                                                                                    \
  hipLaunchKernelGGL((int8_rows_kernel<LANES, R>), dim3((M + 256 / LANES - 1) / (256 / LANES)), dim3(256), 0, stream, codes, scales, \
                     x, x_stride, M, K, padded, clear, clears)
  if (padded <= 512) LI_ROWS(64, 1);
  else if (padded <= 1024) LI_ROWS(64, 2);
  else if (padded <= 2048) LI_ROWS(256, 1);
  else if (padded <= 4096) LI_ROWS(256, 2);
  else if (padded <= 8192) LI_ROWS(256, 4);
  else if (padded <= 16384) LI_ROWS(256, 8);
  else LI_ROWS(256, 0);
#undef LI_ROWS
}

// ---- up to 8 rows of x, in one launch --------------------------------------------------------------

#define LI_UNITS 256       // compute units

#define LF_WAVES 8
#define LF_ROWS 8

// A workgroup takes 16 rows of W (16 of gate and 16 of up), a wave an eighth of K: everything it reads is on its way from its
// first instructions on, x first, since loads come back in order. While W comes, the rows' maxima are found (one barrier) and
// each wave makes the codes of its own part of K, which it alone reads. W goes from memory to the registers that the matrix
// cores take it from, NS stages a wave. The waves' sums meet in LDS. R: rows of x, M of which exist; the others are not looked at.
template <int NS, int R, int T, int FORM, bool ONCE>
__global__ void __launch_bounds__(64 * LF_WAVES) linear_int8_few_kernel(void* __restrict__ out, const bf16_t* __restrict__ x,
                                                                       int64_t x_stride, const int8_t* __restrict__ w,
                                                                       const float* __restrict__ ws, const bf16_t* __restrict__ bias,
                                                                       int M, int N, int K) {
  constexpr bool GATED = FORM == LI_SILU;
  constexpr int V = (NS + 3) / 4, ROW = NS * LI_STAGE + 16;   // 16: rows at different banks
  constexpr int CODES = LF_WAVES * R * ROW, SUMS = LF_WAVES * T * 1024;
  __shared__ __attribute__((aligned(16))) char smem[CODES > SUMS ? CODES : SUMS];
  __shared__ __attribute__((aligned(16))) uint32_t tops[(R + 1) / 2][LF_WAVES];
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int columns = GATED ? N / 2 : N, n0 = blockIdx.x * (GATED ? 16 : 16 * T);
  const int stages_all = (K + LI_STAGE - 1) / LI_STAGE;
  const int first = stages_all * wave / LF_WAVES, stages = stages_all * (wave + 1) / LF_WAVES - first, k0 = first * LI_STAGE;
  constexpr uint32_t NOWHERE = 0x7fffffffu;        // behind every range: zeros
  u16x8 v[R][V];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const auto row = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t*>(x + (int64_t)min(r, M - 1) * x_stride), 0, K * 2, 0x00020000);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = lane + j * 64;
      v[r][j] = __builtin_bit_cast(u16x8, __builtin_amdgcn_raw_buffer_load_b128(row, i < stages * 16 ? (k0 + i * 8) * 2 : NOWHERE, 0, 0));
    }
  }
  u32x4 b[T][NS][2];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const auto rows = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(w + (int64_t)min(n0 + t * (GATED ? columns : 16), N - 16) * K), 0, 16 * K,
                                                           0x00020000);
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        b[t][s][ks] = __builtin_amdgcn_raw_buffer_load_b128(rows, s < stages ? col * K + k0 + s * LI_STAGE + ks * 64 + grp * 16 : NOWHERE, 0,
                                                            ONCE ? 2 : 0);
  }
  __builtin_amdgcn_sched_barrier(0);
  // two rows' maxima side by side
  uint32_t top[(R + 1) / 2];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    u16x8 m = v[r][0] & (u16x8)(unsigned short)0x7fff;
#pragma unroll
    for (int j = 1; j < V; ++j) m = __builtin_elementwise_max(m, v[r][j] & (u16x8)(unsigned short)0x7fff);
    uint32_t of = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) of = max(of, (uint32_t)m[j]);
    top[r >> 1] = r & 1 ? top[r >> 1] | of << 16 : of;
  }
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int p = 0; p < (R + 1) / 2; ++p) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
      top[p] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top[p]),
                                                                     __builtin_bit_cast(u16x2, __shfl_xor(top[p], off))));
    if (lane == 0) tops[p][wave] = top[p];
  }
  // not __syncthreads: what is on its way from memory does not have to have come
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  // lane r has row r's scale
  u16x2 most = {};
#pragma unroll
  for (int e = 0; e < LF_WAVES; ++e) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, tops[min((lane & 7) >> 1, (R + 1) / 2 - 1)][e]));
  const Int8Row mine(lane & 1 ? most[1] : most[0]);
  char* codes = smem + wave * (R * ROW);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= M) continue;
    Int8Row by = mine;
    by.up = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine.up), r));
    by.most = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine.most), r));
    by.inverse = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine.inverse), r));
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = lane + j * 64;
      if (NS % 4 == 0 || i < NS * 16) *reinterpret_cast<u32x2*>(codes + r * ROW + i * 8) = by.codes(v[r][j]);
    }
  }
  // this wave's own part of LDS: in order, only the compiler is held
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  i32x4 acc[T];
#pragma unroll
  for (int t = 0; t < T; ++t) acc[t] = i32x4{0, 0, 0, 0};
  const char* of = codes + min(col, M - 1) * ROW + grp * 16;
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const i32x4 c = *reinterpret_cast<const i32x4*>(of + s * LI_STAGE + ks * 64);
#pragma unroll
      for (int t = 0; t < T; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, b[t][s][ks]), c, acc[t], 0, 0, 0);
    }
  __syncthreads();                                 // the codes are done with
#pragma unroll
  for (int t = 0; t < T; ++t) reinterpret_cast<i32x4*>(smem)[(t * LF_WAVES + wave) * 64 + lane] = acc[t];
  const float s = __shfl(mine.scale, col & 7);
  __syncthreads();
  if (wave > 0 || col >= M) return;
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int e = 1; e < LF_WAVES; ++e) acc[t] += reinterpret_cast<const i32x4*>(smem)[(t * LF_WAVES + e) * 64 + lane];
  f32x4 y[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int n = min(n0 + t * (GATED ? columns : 16), N - 16) + grp * 4;
    const f32x4 by = *reinterpret_cast<const f32x4*>(ws + n);
#pragma unroll
    for (int r = 0; r < 4; ++r) y[t][r] = (float)acc[t][r] * s * by[r];
    if (FORM == LI_BF16 && bias) {
      const bf16x4_vec add = *reinterpret_cast<const bf16x4_vec*>((const short*)bias + n);
#pragma unroll
      for (int r = 0; r < 4; ++r) y[t][r] += bf16_to_f32(add[r]);
    }
  }
  if constexpr (GATED) {
#pragma unroll
    for (int r = 0; r < 4; ++r) y[0][r] = y[0][r] / (1.0f + __expf(-y[0][r])) * y[1][r];
  }
#pragma unroll
  for (int t = 0; t < (GATED ? 1 : T); ++t) {
    const int n = n0 + t * 16 + grp * 4;
    if (n >= columns) continue;
    if constexpr (FORM == LI_PART)
      *reinterpret_cast<f32x4*>((float*)out + (int64_t)col * N + n) = y[t];
    else
      *reinterpret_cast<bf16x4_vec*>((short*)out + (int64_t)col * columns + n) = tp_pack(y[t][0], y[t][1], y[t][2], y[t][3]);
  }
}

struct Int8Few {
  int ns, tiles;             // stages of a wave, 0 where a product goes the way of two launches; tiles of 16 rows of W
};

// Two tiles where one each makes more workgroups than compute units, but no more than twice as many: half as often are the
// codes made (6144 x 4096, 5 rows: 9.4 us, 10.3 with one; 8 rows 10.6 and 11.9). Deeper products have no registers for that.
//
// Each workgroup makes the codes anew. In one round of workgroups that is hidden for long; in more the way of two launches, which
// streams W a little faster, catches up. us of two launches and so:
//   one round   4096 x 4096   1 row 11.4, 5.9   8 rows 11.6, 8.3     1024 x 4096   1 row 9.7, 4.7   8 rows 9.8, 7.4     1152 x 896   5 rows 7.2, 5.6
//               4096 x 14336  1 row 19.0, 14.0   4 rows 19.7, 18.1     896 x 4864   6 rows 10.1, 9.7   8 rows 10.2, 10.4
//   two         9728 x 896 gated   4 rows 8.0, 7.5   5 rows 7.9, 9.1     8192 x 8192   4 rows 19.2, 16.7   5 rows 19.5, 20.8
//   four        16384 x 4096   4 rows 17.3, 16.3   6 rows 17.5, 18.0     28672 x 4096 gated   1 row 26.4, 25.1   5 rows 26.3, 27.9
//               13824 x 5120   1 row 18.8, 17.1   2 rows 18.8, 20.2
//   eight       32768 x 4096   3 rows 27.6, 26.8   5 rows 27.6, 30.6
static Int8Few int8_few(int M, int N, int K, int form) {
  if (M > LF_ROWS) return {0, 0};
  const int stages = (K + LI_STAGE * LF_WAVES - 1) / (LI_STAGE * LF_WAVES), most = form == LI_SILU ? 4 : M <= 4 ? 16 : 8;   // by registers
  if (stages > most) return {0, 0};
  const int ns = stages <= 2 ? 2 : stages <= 4 ? 4 : stages <= 8 ? 8 : 16, steps = (ns + 3) / 4;
  const int tiles = form == LI_SILU || (N > 16 * LI_UNITS && N <= 32 * LI_UNITS && ns <= 4) ? 2 : 1;
  const int64_t rounds = (N / 16 + (int64_t)tiles * LI_UNITS - 1) / ((int64_t)tiles * LI_UNITS);
  if (rounds == 1 ? M * steps > 16 : M > 4 || rounds * steps * steps > 8) return {0, 0};
  return {ns, tiles};
}

extern "C" bool linear_int8_few(int M, int N, int K, int form) { return int8_few(M, N, K, form).ns > 0; }

#define LI_ONCE (8 << 20)
#define LI_ONCE_ALONE ((int64_t)320 << 20)

template <int NS, int R, int T, int FORM>
static int linear_int8_few_go(void* out, const bf16_t* x, int64_t x_stride, const int8_t* w, const float* ws, const bf16_t* bias, int M, int N,
                              int K, bool once, hipStream_t stream) {
  const dim3 grid(FORM == LI_SILU ? N / 32 : (N / 16 + T - 1) / T), block(64 * LF_WAVES);
  if (once)
    hipLaunchKernelGGL((linear_int8_few_kernel<NS, R, T, FORM, true>), grid, block, 0, stream, out, x, x_stride, w, ws, bias, M, N, K);
  else
    hipLaunchKernelGGL((linear_int8_few_kernel<NS, R, T, FORM, false>), grid, block, 0, stream, out, x, x_stride, w, ws, bias, M, N, K);
  return 0;
}

// as launch_linear_int8, of x itself; linear_int8_few says whether it may
extern "C" int launch_linear_int8_few(void* out, const bf16_t* x, int64_t x_stride, const int8_t* w, const float* ws, const bf16_t* bias, int M,
                                      int N, int K, int form, bool once, hipStream_t stream) {
  const int64_t bytes = (int64_t)N * K;
  once = once ? bytes >= LI_ONCE : bytes >= LI_ONCE_ALONE;
  const auto [ns, tiles] = int8_few(M, N, K, form);
  // rows that are not there are loaded and looked at all the same, so there is a form of 6 of the depth that most matrices have (K of
  // 2049 to 4096). us with 8 and 6 rows, of 5 and of 6: 1024 x 4096 6.0 5.6, 6.3 5.9; 2560 x 2560 6.1 5.7, 6.4 5.9; 4096 x 4096 7.4 7.1,
  // 7.6 7.4; 8192 x 4096 10.8 10.4, 11.0 10.7
#define LF_CASE(NS, R)                                                                                                             \
  if (ns == NS && M <= R) {                                                                                                        \
    if constexpr (NS <= 4) {                                                                                                       \
      if (form == LI_BF16 && tiles == 2) return linear_int8_few_go<NS, R, 2, LI_BF16>(out, x, x_stride, w, ws, bias, M, N, K, once, stream); \
      if (form == LI_PART && tiles == 2) return linear_int8_few_go<NS, R, 2, LI_PART>(out, x, x_stride, w, ws, bias, M, N, K, once, stream); \
    }                                                                                                                              \
    if (form == LI_BF16) return linear_int8_few_go<NS, R, 1, LI_BF16>(out, x, x_stride, w, ws, bias, M, N, K, once, stream);       \
    if (form == LI_PART) return linear_int8_few_go<NS, R, 1, LI_PART>(out, x, x_stride, w, ws, bias, M, N, K, once, stream);       \
    if constexpr (NS <= 4) return linear_int8_few_go<NS, R, 2, LI_SILU>(out, x, x_stride, w, ws, bias, M, N, K, once, stream);     \
  }
  LF_CASE(2, 1)
  LF_CASE(2, 4)
  LF_CASE(2, 8)
  LF_CASE(4, 1)
  LF_CASE(4, 4)
  LF_CASE(4, 6)
  LF_CASE(4, 8)
  LF_CASE(8, 1)
  LF_CASE(8, 4)
  LF_CASE(8, 8)
  LF_CASE(16, 1)
  LF_CASE(16, 4)
#undef LF_CASE
  return -1;
}

// ---- few rows or columns -------------------------------------------------------------------------

// linear_rows_kernel of whole numbers. K, padded: bytes of a row of w and of x. PART leaves fp32 sums [splits, M, N], the
// others add their shares up (part, count) and write bf16.
template <int NI, int MJ, int FORM, int KB, bool ONCE>
__global__ void __launch_bounds__(TP_THREADS, 1) linear_int8_rows_kernel(
    void* __restrict__ out, const int8_t* __restrict__ x, const float* __restrict__ xs, const int8_t* __restrict__ w,
    const float* __restrict__ ws, const bf16_t* __restrict__ bias, float* __restrict__ part, int* __restrict__ count, int M, int N,
    int K, int padded, int m_tiles, int splits) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  constexpr bool GATED = FORM == LI_SILU;
  constexpr int BN = GATED ? 16 * NI : 32 * NI;    // columns of the result
  const int columns = GATED ? N / 2 : N;
  const int n_tiles = (columns + BN - 1) / BN, all = n_tiles * splits * m_tiles, xcd = blockIdx.x & 7;
  const int begin = (int)((int64_t)all * xcd >> 3), items = (int)((int64_t)all * (xcd + 1) >> 3) - begin;
  const int at = blockIdx.x >> 3;
  if (at >= items) return;
  const int item = begin + at, rest = item / m_tiles, share = rest / n_tiles, n0 = rest % n_tiles * BN;
  const int rows = (M + m_tiles - 1) / m_tiles;    // even parts
  const int m0 = item % m_tiles * rows, m_end = min(M, m0 + rows);
  const int stages_all = padded / LI_STAGE, first = (int)((int64_t)stages_all * share / splits);
  const int stages = (int)((int64_t)stages_all * (share + 1) / splits) - first, k0 = first * LI_STAGE;
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  i32x4 acc[NI][MJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  // W rows of a gated tile: 8 * NI gate, the same of up, the next gate, their up
  const int n_put = GATED ? n0 + (wave >> 1) * (8 * NI) : n0 + wave * (8 * NI);
  const bf16_t* wk = reinterpret_cast<const bf16_t*>(w + (GATED ? (int64_t)(wave & 1) * columns : 0) * K + k0);
  const TileRows xr(reinterpret_cast<const bf16_t*>(x + k0), m0 + wave * MJ * 8, m_end, MJ * 8, padded / 2, (padded - k0) / 2, lane);
  const TileRowsOf<ONCE> wr(wk, n_put, columns, 8 * NI, K / 2, (K - k0) / 2, lane);
  tile_product<MJ, NI, KB * 1024>(acc, wr, xr, stages, stages * xcd / 8, smem);
  if constexpr (FORM != LI_PART) {
    if (splits > 1) {
      const int tile = rest % n_tiles * m_tiles + item % m_tiles;
      if (!tile_fold<MJ>(acc, part + (int64_t)tile * splits * (NI * MJ * TP_THREADS * 4), share, splits, count + tile, smem)) return;
    }
  }
  const int m = m0 + (wave & 1) * MJ * 16 + col, n = n0 + (wave >> 1) * (BN / 2) + grp * 4;
#pragma unroll
  for (int j = 0; j < MJ; ++j) {
    const int mr = m + j * 16;
    if (mr >= m_end) continue;
    const float s = xs[mr];
#pragma unroll
    for (int i = 0; i < (GATED ? NI / 2 : NI); ++i) {
      const int nc = n + i * 16;
      if (nc >= columns) continue;
      const f32x4 t = *reinterpret_cast<const f32x4*>(ws + nc);
      f32x4 v;
      if constexpr (GATED) {
        const f32x4 tu = *reinterpret_cast<const f32x4*>(ws + columns + nc);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float g = (float)acc[i][j][r] * s * t[r], u = (float)acc[i + NI / 2][j][r] * s * tu[r];
          v[r] = g / (1.0f + __expf(-g)) * u;
        }
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = (float)acc[i][j][r] * s * t[r];
      }
      if constexpr (FORM == LI_PART) {
        *reinterpret_cast<f32x4*>((float*)out + ((int64_t)share * M + mr) * N + nc) = v;
      } else {
        if (FORM == LI_BF16 && bias) {
          const bf16x4_vec b = *reinterpret_cast<const bf16x4_vec*>((const short*)bias + nc);
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] += bf16_to_f32(b[r]);
        }
        *reinterpret_cast<bf16x4_vec*>((short*)out + (int64_t)mr * columns + nc) = tp_pack(v[0], v[1], v[2], v[3]);
      }
    }
  }
}


// Which kernel a product goes to: ni 2 or 4, tiles of 64 or 128 rows of W by 32 * mj of x, shared out over K; ni 8, tiles of 256
// by 32 * mj, the last round of them in shares or not.
struct Int8Plan {
  int ni, mj, m_tiles, splits;
};

// us of a stage: of a workgroup that has a compute unit to itself, and of two that share one (160 KB of LDS hold two of those
// with 80); [ni / 4][mj]
static const double LI_ALONE[2][5] = {{0, 0.16, 0.22, 0.27, 0.32}, {0, 0, 0.32, 0.43, 0.58}};
static const double LI_PAIR[2][5] = {{0, 0.38, 0.38, 0.46, 0.49}, {0, 0, 0.57, 0, 0}};
static const double LI_TILE[9] = {0, 0, 0.42, 0.60, 0.72, 0.87, 1.0, 1.2, 1.3};   // of tiles of 256

static constexpr int li_ring(int ni, int mj) { return ni == 2 || mj <= 2 ? 80 : 160; }   // KB

// The tiles that take the least time by what rounds of compute units, stages, the stream of W, reads through the caches and
// sums through memory take. The constants are fitted to 4500 measured products, 10 matrices of 1024 x 4096 to 28672 x 4096 by 1
// to 2100 rows in all tiles; what they pick is 0.5% behind the best tiles on average, 11% at most. With tiles of 64 rows of W
// and 32 * ceil(M / 32) of x up to 128 rows and those of 256 above: 4608 x 3584, 333 rows, 29.7 us and so 21.9; 2048 x 2048,
// 128 rows, 15.5 and 11.2; 4096 x 4096, 512 rows, 34.7 and 22.
static Int8Plan int8_plan(int64_t M, int64_t N, int64_t K, int form) {
  const bool gated = form == LI_SILU;
  const int64_t columns = gated ? N / 2 : N, stages = int8_rows_padded((int)K) / LI_STAGE;
  const double stream = (double)N * K / 5.1e6;
  Int8Plan best = {2, 1, 1, 1};
  double least = 1e300;
  for (int ni = 2; ni <= 4; ni += 2)
    for (int mj = M <= 32 ? 1 : 2; mj <= (M <= 32 ? 1 : 4); ++mj) {
      if (ni == 4 && mj == 1) continue;
      const int64_t m_tiles = (M + 32 * mj - 1) / (32 * mj), wide = (gated ? 16 : 32) * ni;
      if (mj > 2 && M <= 32 * (mj - 1)) continue;
      if (form == LI_PART && m_tiles > LI_UNITS) continue;
      const int64_t tiles = m_tiles * ((columns + wide - 1) / wide);
      for (int64_t splits = 1; splits <= 8 && (splits == 1 || (splits * 3 <= stages && tiles * splits <= 600)); ++splits) {
        const double deep = (double)((stages + splits - 1) / splits);
        const int64_t of_unit = (tiles * splits + LI_UNITS - 1) / LI_UNITS;
        const double run = li_ring(ni, mj) == 80
                               ? (double)(of_unit / 2) * LI_PAIR[ni / 4][mj] * deep + (double)(of_unit % 2) * LI_ALONE[ni / 4][mj] * deep +
                                     4.0 * (double)((of_unit + 1) / 2)
                               : (double)of_unit * (LI_ALONE[ni / 4][mj] * deep + 4.0);
        const double cost = (run > stream ? run : stream) + (double)(tiles * splits) * deep * (ni + mj) * 4096 / 44e6 +
                            (splits > 1 ? 0.5 + 0.21 * (double)(ni * mj * splits) : 0.0);
        if (cost < least) least = cost, best = {ni, mj, (int)m_tiles, (int)splits};
      }
    }
  if (form == LI_PART || M <= 128) return best;
  const int64_t n_tiles = (columns + (gated ? 127 : 255)) / (gated ? 128 : 256);
  for (int mj = 8; mj >= 2; --mj) {
    const int64_t m_tiles = (M + 32 * mj - 1) / (32 * mj), tiles = m_tiles * n_tiles, unit = (tiles + 7) / 8, rest = unit % TP_SLOTS;
    const double round = LI_TILE[mj] * (double)stages + 5.9, reads = (double)(tiles * stages) * (8 + mj) * 4096 / 44e6;
    const double whole = (double)((unit + TP_SLOTS - 1) / TP_SLOTS) * round;
    if ((whole > stream ? whole : stream) + reads < least)
      least = (whole > stream ? whole : stream) + reads, best = {8, mj, (int)m_tiles, 1};
    if (stages < 16 || rest == 0 || rest > TP_SLOTS / 2) continue;
    int64_t shares = TP_SLOTS / rest < TP_SHARES ? TP_SLOTS / rest : TP_SHARES;
    shares = shares < stages / 8 ? shares : stages / 8;
    const double shared = (double)(unit / TP_SLOTS) * round + LI_TILE[mj] * (double)stages / (double)shares + 10 + 0.48 * (double)(mj * shares);
    if ((shared > stream ? shared : stream) + reads < least)
      least = (shared > stream ? shared : stream) + reads, best = {8, mj, (int)m_tiles, (int)shares};
  }
  return best;
}

// shares of form 2 of a product whose codes are made before it
extern "C" int linear_int8_splits(int M, int N, int K) { return int8_plan(M, N, K, LI_PART).splits; }

template <int NI, int MJ, int FORM, bool ONCE>
static int linear_int8_rows_go(const Int8Plan& p, void* out, const int8_t* x, const float* xs, const int8_t* w, const float* ws,
                               const bf16_t* bias, float* part, int* count, int M, int N, int K, hipStream_t stream) {
  constexpr int KB = li_ring(NI, MJ), BN = (FORM == LI_SILU ? 16 : 32) * NI;
  if (!tp_lds_ready(reinterpret_cast<const void*>(linear_int8_rows_kernel<NI, MJ, FORM, KB, ONCE>))) return -1;
  constexpr int LDS = TileRing<MJ, NI, KB * 1024>::STRIDE * TileRing<MJ, NI, KB * 1024>::RING;
  const int64_t all = (int64_t)(((FORM == LI_SILU ? N / 2 : N) + BN - 1) / BN) * p.splits * p.m_tiles;
  hipLaunchKernelGGL((linear_int8_rows_kernel<NI, MJ, FORM, KB, ONCE>), dim3((all + 7) / 8 * 8), dim3(TP_THREADS), LDS, stream, out, x, xs,
                     w, ws, bias, part, count, M, N, K, int8_rows_padded(K), p.m_tiles, p.splits);
  return 0;
}

template <int FORM>
static int linear_int8_rows_form(const Int8Plan& p, void* out, const int8_t* x, const float* xs, const int8_t* w, const float* ws,
                                 const bf16_t* bias, float* part, int* count, int M, int N, int K, bool once, hipStream_t stream) {
  const int64_t bytes = (int64_t)N * K;
  once = p.m_tiles == 1 && (once ? bytes >= LI_ONCE : bytes >= LI_ONCE_ALONE);   // row tiles read W one after the other
#define LI_CASE(NI, MJ)                                                                                                           \
  if (p.ni == NI && p.mj == MJ)                                                                                                   \
    return once ? linear_int8_rows_go<NI, MJ, FORM, true>(p, out, x, xs, w, ws, bias, part, count, M, N, K, stream)               \
                : linear_int8_rows_go<NI, MJ, FORM, false>(p, out, x, xs, w, ws, bias, part, count, M, N, K, stream)
  LI_CASE(2, 1);
  LI_CASE(2, 2);
  LI_CASE(2, 3);
  LI_CASE(2, 4);
  LI_CASE(4, 2);
  LI_CASE(4, 3);
  LI_CASE(4, 4);
#undef LI_CASE
  return -1;
}

// ---- large products ------------------------------------------------------------------------------

#define LI_BAND 8          // row tiles of a band

template <int ACT, int MJ>
__global__ void __launch_bounds__(TP_THREADS, 1) linear_int8_tiles_kernel(
    bf16_t* __restrict__ out, const int8_t* __restrict__ x, const float* __restrict__ xs, const int8_t* __restrict__ w,
    const float* __restrict__ ws, const bf16_t* __restrict__ bias, float* __restrict__ part, int* __restrict__ count, int M, int N, int K,
    int padded, int m_tiles) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  constexpr int BN = ACT ? 128 : 256;              // output columns of a workgroup
  const int n_tiles = (N + BN - 1) / BN;
  // an XCD's tiles are neighbours, in bands of rows and column by column in them
  const int xcd = blockIdx.x & 7;
  const int all = m_tiles * n_tiles;
  const int begin = (int)((int64_t)all * xcd / 8), tiles = (int)((int64_t)all * (xcd + 1) / 8) - begin;
  const int stages_all = padded / LI_STAGE;
  const TileShare sh(blockIdx.x >> 3, tiles, stages_all, part, count, xcd, 256 * 32 * MJ);
  if (sh.tile >= tiles) return;
  const int tile = begin + sh.tile;
  const int bands = (m_tiles + LI_BAND - 1) / LI_BAND, deep = (m_tiles + bands - 1) / bands;
  const int band = tile / (deep * n_tiles), in = tile % (deep * n_tiles);
  const int high = min(deep, m_tiles - band * deep);
  const int rows = (M + m_tiles - 1) / m_tiles;    // even parts
  const int m0 = (band * deep + in % high) * rows, m_end = min(M, m0 + rows);
  const int n0 = in / high * BN;
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  i32x4 acc[8][MJ];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  const int stages = sh.length(stages_all), k0 = sh.first(stages_all) * LI_STAGE;
  const int m = m0 + (wave & 1) * MJ * 16;         // first row of this wave's results
  const TileRows xr(reinterpret_cast<const bf16_t*>(x + k0), m0 + wave * MJ * 8, m_end, MJ * 8, padded / 2, (padded - k0) / 2, lane);
  // W rows of a gated tile: 64 gate, 64 up, the next 64 gate, 64 up
  const int n_put = ACT ? n0 + (wave >> 1) * 64 : n0 + wave * 64;
  const TileRows wr(reinterpret_cast<const bf16_t*>(w + (ACT ? (int64_t)(wave & 1) * N : 0) * K + k0), n_put, N, 64, K / 2, (K - k0) / 2, lane);
  tile_product<MJ>(acc, wr, xr, stages, stages * xcd / 8, smem);
  if (sh.shares > 1 && !tile_fold<MJ>(acc, sh.part, sh.share, sh.shares, sh.count, smem)) return;
  float s[MJ];
#pragma unroll
  for (int j = 0; j < MJ; ++j) s[j] = xs[min(m + j * 16 + col, M - 1)];
  const int n = n0 + (wave >> 1) * (ACT ? 64 : 128);
  // scales and bias of 4 columns: N is a multiple of 16, what is behind it is not stored
  auto of = [&](int at) { return *reinterpret_cast<const f32x4*>(ws + (ACT && at >= 2 * N ? 0 : !ACT && at >= N ? 0 : at)); };
  if constexpr (ACT) {
    tile_store<4, MJ>(out + (int64_t)m * N + n, N, m_end - m, N - n, smem, [&](int i, int j) {
      const int c = min(n + i * 16 + grp * 4, N - 4);
      const f32x4 tg = of(c), tu = of(N + c);
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float g = (float)acc[i][j][r] * s[j] * tg[r], u = (float)acc[i + 4][j][r] * s[j] * tu[r];
        v[r] = g / (1.0f + __expf(-g)) * u;
      }
      return tp_pack(v[0], v[1], v[2], v[3]);
    });
  } else {
    tile_store<8, MJ>(out + (int64_t)m * N + n, N, m_end - m, N - n, smem, [&](int i, int j) {
      const int c = min(n + i * 16 + grp * 4, N - 4);
      const f32x4 t = of(c);
      bf16x4_vec b = {0, 0, 0, 0};
      if (bias) b = *reinterpret_cast<const bf16x4_vec*>((const short*)bias + c);
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = (float)acc[i][j][r] * s[j] * t[r] + bf16_to_f32(b[r]);
      return tp_pack(v[0], v[1], v[2], v[3]);
    });
  }
}

template <int ACT, int MJ>
static int linear_int8_tiles_go(void* out, const int8_t* x, const float* xs, const int8_t* w, const float* ws, const bf16_t* bias,
                                float* part, int* count, int M, int N, int K, hipStream_t stream) {
  if (!tp_lds_ready(reinterpret_cast<const void*>(linear_int8_tiles_kernel<ACT, MJ>))) return -1;
  constexpr int BN = ACT ? 128 : 256;
  const int m_tiles = (M + 32 * MJ - 1) / (32 * MJ);
  const int64_t all = (int64_t)m_tiles * ((N + BN - 1) / BN);
  hipLaunchKernelGGL((linear_int8_tiles_kernel<ACT, MJ>), dim3(((all + 7) / 8 + (part ? TP_SLOTS : 0)) * 8), dim3(TP_THREADS), TP_LDS, stream,
                     (bf16_t*)out, x, xs, w, ws, bias, part, count, M, N, K, int8_rows_padded(K), m_tiles);
  return 0;
}

// ---- the calls -----------------------------------------------------------------------------------

// floats of part and zeros of count that a product (form 0 or 1; N: rows of w) takes, 0 where it has no shares
extern "C" int64_t linear_int8_room(int M, int N, int K, int form, int* zeros) {
  *zeros = 0;
  const Int8Plan p = int8_plan(M, N, K, form);
  if (p.splits == 1) return 0;
  if (p.ni == 8) {
    *zeros = LI_UNITS;
    return (int64_t)LI_UNITS * 256 * 32 * p.mj;
  }
  const int wide = (form == LI_SILU ? 16 : 32) * p.ni;
  const int64_t tiles = (int64_t)p.m_tiles * (((form == LI_SILU ? N / 2 : N) + wide - 1) / wide);
  *zeros = (int)tiles;
  return tiles * p.splits * (p.ni * p.mj * TP_THREADS * 4);
}

// form 0: bf16 [M, N] (+ bias), 1: silu(gate) * up bf16 [M, N / 2]; 2: fp32 sums [splits, M, N] of up to 128 rows. part and
// count (zeroed): of linear_int8_room. 0, or -1 where the LDS cannot be had.
extern "C" int launch_linear_int8(void* out, const int8_t* x, const float* xs, const int8_t* w, const float* ws, const bf16_t* bias,
                                  float* part, int* count, int M, int N, int K, int form, bool once, hipStream_t stream) {
  const Int8Plan p = int8_plan(M, N, K, form);
  if (p.ni < 8)
    return form == LI_SILU   ? linear_int8_rows_form<LI_SILU>(p, out, x, xs, w, ws, bias, part, count, M, N, K, once, stream)
           : form == LI_PART ? linear_int8_rows_form<LI_PART>(p, out, x, xs, w, ws, bias, part, count, M, N, K, once, stream)
                             : linear_int8_rows_form<LI_BF16>(p, out, x, xs, w, ws, bias, part, count, M, N, K, once, stream);
  const bool gated = form == LI_SILU;
  const int n = gated ? N / 2 : N;
#define LI_CASE(MJ)                                                                                                 \
  case MJ:                                                                                                          \
    return gated ? linear_int8_tiles_go<1, MJ>(out, x, xs, w, ws, bias, part, count, M, n, K, stream)               \
                 : linear_int8_tiles_go<0, MJ>(out, x, xs, w, ws, bias, part, count, M, n, K, stream)
  switch (p.mj) {
    LI_CASE(2);
    LI_CASE(3);
    LI_CASE(4);
    LI_CASE(5);
    LI_CASE(6);
    LI_CASE(7);
    LI_CASE(8);
    default: return -1;
  }
#undef LI_CASE
}
