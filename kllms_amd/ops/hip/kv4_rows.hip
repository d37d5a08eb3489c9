// Rows into a 4-bit key/value cache and out of it again (kv4.h has the form of a row), for gfx950.
//
// Both are passes over memory: eight threads a row, 16-byte loads and stores of bf16. A row's codes are put together by moves
// between its eight lanes.

#include "kv4.h"

// rows t of k and v [T, G, 128] to slots[t] of the caches [NB, G, block, 64], scales [NB, G, block, 2] words. A slot outside
// the cache is nobody's: its row goes nowhere.
__global__ void __launch_bounds__(256) kv4_store_kernel(const bf16_t* __restrict__ k, const bf16_t* __restrict__ v,
                                                        uint32_t* __restrict__ k_cache, uint32_t* __restrict__ v_cache,
                                                        uint32_t* __restrict__ k_scale, uint32_t* __restrict__ v_scale,
                                                        const int64_t* __restrict__ slots, int64_t n, int G, int64_t k_stride,
                                                        int64_t v_stride, int block_size, int64_t positions) {
  for (int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x; idx < n; idx += (int64_t)gridDim.x * 256) {
    const int piece = (int)(idx & 7);
    const int64_t th = idx >> 3, t = th / (2 * G);
    const int head = (int)(th - t * (2 * G)), g = head < G ? head : head - G;
    const bool is_v = head >= G;
    const short* row = (is_v ? (const short*)v + t * v_stride : (const short*)k + t * k_stride) + g * 128;
    const bf16x8_vec a = *reinterpret_cast<const bf16x8_vec*>(row + piece * 8);
    const bf16x8_vec b = *reinterpret_cast<const bf16x8_vec*>(row + 64 + piece * 8);
    const int64_t slot = slots[t];
    if (slot < 0 || slot >= positions) continue;       // a row's eight lanes as one
    const int64_t at = (slot / block_size * G + g) * block_size + slot % block_size;
    kv4_store_row((is_v ? v_cache : k_cache) + at * (KV4_BYTES / 4), (is_v ? v_scale : k_scale) + at * KV4_GROUPS, piece, a, b);
  }
}

extern "C" void launch_kv4_store(const bf16_t* k, const bf16_t* v, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                                 const int64_t* slots, int T, int G, int64_t k_stride, int64_t v_stride, int block_size,
                                 int64_t positions, hipStream_t stream) {
  const int64_t n = (int64_t)T * G * 16, blocks = (n + 255) / 256;
  hipLaunchKernelGGL(kv4_store_kernel, dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, stream, k, v,
                     (uint32_t*)k_cache, (uint32_t*)v_cache, (uint32_t*)k_scale, (uint32_t*)v_scale, slots, n, G, k_stride, v_stride,
                     block_size, positions);
}

// What the caches' rows at slots[t] stand for, rounded to bf16: k and v [T, G, 128]. Rows of a slot outside the cache are NaN.
// Thread ``piece`` has words 2 piece, 2 piece + 1: two neighbouring values of each of eight runs of 16.
__global__ void __launch_bounds__(256) kv4_load_kernel(bf16_t* __restrict__ k, bf16_t* __restrict__ v,
                                                       const uint32_t* __restrict__ k_cache, const uint32_t* __restrict__ v_cache,
                                                       const uint32_t* __restrict__ k_scale, const uint32_t* __restrict__ v_scale,
                                                       const int64_t* __restrict__ slots, int64_t n, int G, int block_size,
                                                       int64_t positions) {
  for (int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x; idx < n; idx += (int64_t)gridDim.x * 256) {
    const int piece = (int)(idx & 7);
    const int64_t th = idx >> 3, t = th / (2 * G);
    const int head = (int)(th - t * (2 * G)), g = head < G ? head : head - G;
    const bool is_v = head >= G;
    const int64_t slot = slots[t];
    const bool known = slot >= 0 && slot < positions;
    const int64_t at = known ? (slot / block_size * G + g) * block_size + slot % block_size : 0;
    u32x2_kv4 w = {0u, 0u}, s = {0x7fc07fc0u, 0x7fc07fc0u};
    if (known) {
      w = *reinterpret_cast<const u32x2_kv4*>((is_v ? v_cache : k_cache) + at * (KV4_BYTES / 4) + piece * 2);
      s = *reinterpret_cast<const u32x2_kv4*>((is_v ? v_scale : k_scale) + at * KV4_GROUPS);
    }
    short* row = (short*)(is_v ? v : k) + (t * G + g) * 128 + piece * 2;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const uint32_t sc = s[(p & 3) >> 1];
      const short x = f32_to_bf16(__builtin_fmaf((float)(w[0] >> 4 * p & 15), kv4_step(sc), kv4_least(sc)));
      const short y = f32_to_bf16(__builtin_fmaf((float)(w[1] >> 4 * p & 15), kv4_step(sc), kv4_least(sc)));
      *reinterpret_cast<uint32_t*>(row + 32 * (p & 3) + 16 * (p >> 2)) = (uint16_t)x | (uint32_t)(uint16_t)y << 16;
    }
  }
}

extern "C" void launch_kv4_load(bf16_t* k, bf16_t* v, const void* k_cache, const void* v_cache, const void* k_scale,
                                const void* v_scale, const int64_t* slots, int T, int G, int block_size, int64_t positions,
                                hipStream_t stream) {
  const int64_t n = (int64_t)T * G * 16, blocks = (n + 255) / 256;
  hipLaunchKernelGGL(kv4_load_kernel, dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, stream, k, v,
                     (const uint32_t*)k_cache, (const uint32_t*)v_cache, (const uint32_t*)k_scale, (const uint32_t*)v_scale, slots, n, G,
                     block_size, positions);
}
