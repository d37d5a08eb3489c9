// Rows into a 4-bit key/value cache and out of it again (kv4.h has the form of a row), for gfx950.
//
// Both are passes over memory: eight threads a row, 16-byte loads and stores of bf16. A row's codes are put together by moves
// between its eight lanes. A workgroup has one head of KV4_TOKENS tokens: what it writes of the cache lies together, also the
// scales, of which 16 positions share a line (with all heads of two tokens to a workgroup the parts of a line came from eight
// L2s).
//
// What bounds them: memory, and beside it on the way in the vector units (290 instructions for 16 values). Measured, 8 heads, us in and
// back out: 120 tokens 2.9, 2.7 (a launch); 7777 10.8, 10.7 (41 MB each); 30000 41.9, 28.4.

#include "kv4.h"

#define KV4_TOKENS 32

typedef __bf16 bf16x8_kv4 __attribute__((ext_vector_type(8)));
typedef float f32x8_kv4 __attribute__((ext_vector_type(8)));

// Row of a position in [NB, G, block]; a cache has fewer than 2^31, and a division of 32 bits is a fifth of one of 64
__device__ __forceinline__ int64_t kv4_row_of(int64_t slot, int G, int g, int block_size) {
  const uint32_t block = (uint32_t)slot / (uint32_t)block_size;
  return ((int64_t)block * G + g) * block_size + (uint32_t)slot % (uint32_t)block_size;
}

// rows t of k and v [T, G, 128] to slots[t] of the caches [NB, G, block, 64], scales [NB, G, block, 2] words. A slot outside
// the cache is nobody's: its row goes nowhere.
__global__ void __launch_bounds__(256) kv4_store_kernel(const bf16_t* __restrict__ k, const bf16_t* __restrict__ v,
                                                        uint32_t* __restrict__ k_cache, uint32_t* __restrict__ v_cache,
                                                        uint32_t* __restrict__ k_scale, uint32_t* __restrict__ v_scale,
                                                        const int64_t* __restrict__ slots, int T, int G, int64_t k_stride,
                                                        int64_t v_stride, int block_size, int64_t positions) {
  const int piece = threadIdx.x & 7;
  const int head = blockIdx.x % (2 * G), g = head < G ? head : head - G;
  const bool is_v = head >= G;
  const int64_t t = (int64_t)(blockIdx.x / (2 * G)) * KV4_TOKENS + (threadIdx.x >> 3);
  if (t >= T) return;                                  // a row's eight lanes as one
  const short* row = (is_v ? (const short*)v + t * v_stride : (const short*)k + t * k_stride) + g * 128;
  const bf16x8_vec a = *reinterpret_cast<const bf16x8_vec*>(row + piece * 8);
  const bf16x8_vec b = *reinterpret_cast<const bf16x8_vec*>(row + 64 + piece * 8);
  const int64_t slot = slots[t];
  if (slot < 0 || slot >= positions) return;
  const int64_t at = kv4_row_of(slot, G, g, block_size);
  kv4_store_row((is_v ? v_cache : k_cache) + at * (KV4_BYTES / 4), (is_v ? v_scale : k_scale) + at * KV4_GROUPS, piece, a, b);
}

extern "C" void launch_kv4_store(const bf16_t* k, const bf16_t* v, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                                 const int64_t* slots, int T, int G, int64_t k_stride, int64_t v_stride, int block_size,
                                 int64_t positions, hipStream_t stream) {
  const int64_t blocks = (int64_t)(T / KV4_TOKENS + (T % KV4_TOKENS > 0)) * 2 * G;
  hipLaunchKernelGGL(kv4_store_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, k, v,
                     (uint32_t*)k_cache, (uint32_t*)v_cache, (uint32_t*)k_scale, (uint32_t*)v_scale, slots, T, G, k_stride, v_stride,
                     block_size, positions);
}

// What the caches' rows at slots[t] stand for, rounded to bf16: k and v [T, G, 128]. Rows of a slot outside the cache are NaN.
// Thread ``piece`` has nibble ``piece`` of all words, 16 neighbouring values: a row's 64 bytes are read by eight threads from the
// first-level cache, and written in 16-byte stores (of 4 bytes each, from two words a thread, 7777 rows of 8 heads took 16 us).
__global__ void __launch_bounds__(256) kv4_load_kernel(bf16_t* __restrict__ k, bf16_t* __restrict__ v,
                                                       const uint32_t* __restrict__ k_cache, const uint32_t* __restrict__ v_cache,
                                                       const uint32_t* __restrict__ k_scale, const uint32_t* __restrict__ v_scale,
                                                       const int64_t* __restrict__ slots, int T, int G, int block_size,
                                                       int64_t positions) {
  const int piece = threadIdx.x & 7;
  const int head = blockIdx.x % (2 * G), g = head < G ? head : head - G;
  const bool is_v = head >= G;
  const int64_t t = (int64_t)(blockIdx.x / (2 * G)) * KV4_TOKENS + (threadIdx.x >> 3);
  if (t >= T) return;                                  // a row's eight lanes as one
  const int64_t slot = slots[t];
  const bool known = slot >= 0 && slot < positions;
  const int64_t at = known ? kv4_row_of(slot, G, g, block_size) : 0;
  u32x4_kv4 w[4] = {};
  uint32_t sc = 0x7fc07fc0u;
  if (known) {
    const u32x4_kv4* words = reinterpret_cast<const u32x4_kv4*>((is_v ? v_cache : k_cache) + at * (KV4_BYTES / 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = words[i];
    sc = ((is_v ? v_scale : k_scale) + at * KV4_GROUPS)[(piece & 3) >> 1];
  }
  short* row = (short*)(is_v ? v : k) + (t * G + g) * 128 + 32 * (piece & 3) + 16 * (piece >> 2);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f32x8_kv4 x;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = __builtin_fmaf((float)(w[2 * i + (j >> 2)][j & 3] >> 4 * piece & 15), kv4_step(sc), kv4_least(sc));
    *reinterpret_cast<bf16x8_kv4*>(row + 8 * i) = __builtin_convertvector(x, bf16x8_kv4);
  }
}

extern "C" void launch_kv4_load(bf16_t* k, bf16_t* v, const void* k_cache, const void* v_cache, const void* k_scale,
                                const void* v_scale, const int64_t* slots, int T, int G, int block_size, int64_t positions,
                                hipStream_t stream) {
  const int64_t blocks = (int64_t)(T / KV4_TOKENS + (T % KV4_TOKENS > 0)) * 2 * G;
  hipLaunchKernelGGL(kv4_load_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, k, v,
                     (const uint32_t*)k_cache, (const uint32_t*)v_cache, (const uint32_t*)k_scale, (const uint32_t*)v_scale, slots, T, G,
                     block_size, positions);
}
