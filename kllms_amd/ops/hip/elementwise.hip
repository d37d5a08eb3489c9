// Memory-bound elementwise / normalization kernels for gfx950.
//
// All of these are HBM-bandwidth-bound: the design rules applied are
// G13 (vectorize bf16 as 8-element/16-byte lane loads), G11 (grid-stride with
// a capped grid), and fusion (residual-add folded into RMSNorm; cos/sin for
// RoPE precomputed on host — Appendix B: on-device trig turns memory-bound
// into VALU-bound).

#include "kv4.h"

// --------------------------------------------------------------------------
// RMSNorm: one block per row, row length N (multiple of 8), bf16 in/out.
// y = x / sqrt(mean(x^2) + eps) * w      (fp32 accumulation)
// --------------------------------------------------------------------------
extern "C" __global__ void __launch_bounds__(256) rmsnorm_kernel(
    bf16_t* __restrict__ out, const bf16_t* __restrict__ in,
    const bf16_t* __restrict__ w, int n, float eps) {
  __shared__ float red[16];
  const int row = blockIdx.x;
  const bf16x8_vec* inv = reinterpret_cast<const bf16x8_vec*>(in + (int64_t)row * n);
  bf16x8_vec* outv = reinterpret_cast<bf16x8_vec*>(out + (int64_t)row * n);
  const bf16x8_vec* wv = reinterpret_cast<const bf16x8_vec*>(w);
  const int nvec = n / 8;

  float ss = 0.0f;
  for (int i = threadIdx.x; i < nvec; i += blockDim.x) {
    bf16x8_vec v = inv[i];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float f = bf16_to_f32(v[j]);
      ss += f * f;
    }
  }
  ss = block_reduce_sum<4>(ss, red);
  const float inv_rms = rsqrtf(ss / n + eps);

  for (int i = threadIdx.x; i < nvec; i += blockDim.x) {
    bf16x8_vec v = inv[i];
    bf16x8_vec wv8 = wv[i];
    bf16x8_vec o;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      o[j] = f32_to_bf16(bf16_to_f32(v[j]) * inv_rms * bf16_to_f32(wv8[j]));
    outv[i] = o;
  }
}

// --------------------------------------------------------------------------
// Fused residual-add + RMSNorm: residual += x (written back), y = rmsnorm(residual)
// --------------------------------------------------------------------------
extern "C" __global__ void __launch_bounds__(256) fused_add_rmsnorm_kernel(
    bf16_t* __restrict__ out, const bf16_t* __restrict__ x,
    bf16_t* __restrict__ residual, const bf16_t* __restrict__ w, int n, float eps) {
  __shared__ float red[16];
  const int row = blockIdx.x;
  const bf16x8_vec* xv = reinterpret_cast<const bf16x8_vec*>(x + (int64_t)row * n);
  bf16x8_vec* rv = reinterpret_cast<bf16x8_vec*>(residual + (int64_t)row * n);
  bf16x8_vec* outv = reinterpret_cast<bf16x8_vec*>(out + (int64_t)row * n);
  const bf16x8_vec* wv = reinterpret_cast<const bf16x8_vec*>(w);
  const int nvec = n / 8;

  float ss = 0.0f;
  for (int i = threadIdx.x; i < nvec; i += blockDim.x) {
    bf16x8_vec a = xv[i];
    bf16x8_vec b = rv[i];
    bf16x8_vec s;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float f = bf16_to_f32(a[j]) + bf16_to_f32(b[j]);
      s[j] = f32_to_bf16(f);
      float fs = bf16_to_f32(s[j]);  // accumulate on the bf16-rounded sum
      ss += fs * fs;
    }
    rv[i] = s;
  }
  ss = block_reduce_sum<4>(ss, red);
  const float inv_rms = rsqrtf(ss / n + eps);

  for (int i = threadIdx.x; i < nvec; i += blockDim.x) {
    bf16x8_vec s = rv[i];
    bf16x8_vec wv8 = wv[i];
    bf16x8_vec o;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      o[j] = f32_to_bf16(bf16_to_f32(s[j]) * inv_rms * bf16_to_f32(wv8[j]));
    outv[i] = o;
  }
}

// --------------------------------------------------------------------------
// SwiGLU activation: out = silu(gate) * up, bf16, grid-stride, 8-wide.
// --------------------------------------------------------------------------
extern "C" __global__ void __launch_bounds__(256) silu_mul_kernel(
    bf16_t* __restrict__ out, const bf16_t* __restrict__ gate,
    const bf16_t* __restrict__ up, int64_t nvec, int ncols_vec, int row_stride_vec) {
  // gate/up are [rows, ncols] row-views with a free row stride (the fused
  // gate_up GEMM output), out is contiguous [rows, ncols]
  bf16x8_vec* ov = reinterpret_cast<bf16x8_vec*>(out);
  for (int64_t i = blockIdx.x * blockDim.x + threadIdx.x; i < nvec;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / ncols_vec;
    const int64_t col = i % ncols_vec;
    const int64_t src = row * row_stride_vec + col;
    bf16x8_vec g = reinterpret_cast<const bf16x8_vec*>(gate)[src];
    bf16x8_vec u = reinterpret_cast<const bf16x8_vec*>(up)[src];
    bf16x8_vec o;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float gf = bf16_to_f32(g[j]);
      float s = gf / (1.0f + __expf(-gf));
      o[j] = f32_to_bf16(s * bf16_to_f32(u[j]));
    }
    ov[i] = o;
  }
}

// --------------------------------------------------------------------------
// RoPE (Llama rotate-half): in-place on q [T, H, D] and k [T, KVH, D].
// cos_sin: [max_pos, D] fp32, cos in [0, D/2), sin in [D/2, D).
// Grid: (T, H + KVH); block = D/2 threads (one lane per rotation pair).
// --------------------------------------------------------------------------
extern "C" __global__ void rope_kernel(
    bf16_t* __restrict__ q, bf16_t* __restrict__ k,
    const int64_t* __restrict__ positions, const float* __restrict__ cos_sin,
    int num_q_heads, int num_kv_heads, int head_dim, int q_tstride, int k_tstride) {
  const int t = blockIdx.x;
  const int h = blockIdx.y;
  const int i = threadIdx.x;           // pair index in [0, D/2)
  const int half = head_dim / 2;
  if (i >= half) return;
  const int64_t pos = positions[t];
  const float c = cos_sin[pos * head_dim + i];
  const float s = cos_sin[pos * head_dim + half + i];
  bf16_t* base;
  if (h < num_q_heads) {
    base = q + (int64_t)t * q_tstride + h * head_dim;
  } else {
    base = k + (int64_t)t * k_tstride + (h - num_q_heads) * head_dim;
  }
  float x1 = bf16_to_f32(((const short*)base)[i]);
  float x2 = bf16_to_f32(((const short*)base)[half + i]);
  ((short*)base)[i] = f32_to_bf16(x1 * c - x2 * s);
  ((short*)base)[half + i] = f32_to_bf16(x2 * c + x1 * s);
}

// --------------------------------------------------------------------------
// Paged-KV scatter: k/v [T, KVH, D] -> caches [NB, KVH, BS, D] at flat slots.
// Grid-stride over T*KVH*(D/8); 16-byte lane copies.
// --------------------------------------------------------------------------
extern "C" __global__ void __launch_bounds__(256) store_kv_kernel(
    const bf16_t* __restrict__ k, const bf16_t* __restrict__ v,
    bf16_t* __restrict__ k_cache, bf16_t* __restrict__ v_cache,
    const int64_t* __restrict__ slots, int num_tokens, int kv_heads,
    int head_dim, int block_size, int kv_tstride) {
  const int dvec = head_dim / 8;
  const int64_t total = (int64_t)num_tokens * kv_heads * dvec;
  for (int64_t idx = blockIdx.x * blockDim.x + threadIdx.x; idx < total;
       idx += (int64_t)gridDim.x * blockDim.x) {
    const int dv = idx % dvec;
    const int g = (idx / dvec) % kv_heads;
    const int t = idx / ((int64_t)dvec * kv_heads);
    const int64_t slot = slots[t];
    const int64_t blk = slot / block_size;
    const int off = slot % block_size;
    const bf16x8_vec* src_k =
        reinterpret_cast<const bf16x8_vec*>(k + (int64_t)t * kv_tstride + g * head_dim) + dv;
    const bf16x8_vec* src_v =
        reinterpret_cast<const bf16x8_vec*>(v + (int64_t)t * kv_tstride + g * head_dim) + dv;
    int64_t dst_off = ((blk * kv_heads + g) * block_size + off) * head_dim;
    reinterpret_cast<bf16x8_vec*>(k_cache + dst_off)[dv] = *src_k;
    reinterpret_cast<bf16x8_vec*>(v_cache + dst_off)[dv] = *src_v;
  }
}

// fp8 (e4m3) variant of the paged-KV scatter with PER-ROW dequant scales:
// one 64-lane wave per (token, kv_head) row computes s = max(amax|row|/448,
// 1e-8) over the row's K (and V) values, stores the scales to
// k_scale/v_scale [NB, KVH, BS] and quantizes x/s into the 1-byte caches —
// outlier rows in real checkpoints no longer saturate e4m3's +-448 range.
// T*KVH rows per call is tiny next to the attention reads, so a plain
// strided (non-vectorized) load pattern is fine here.
extern "C" __global__ void __launch_bounds__(256) store_kv_fp8_kernel(
    const bf16_t* __restrict__ k, const bf16_t* __restrict__ v,
    unsigned char* __restrict__ k_cache, unsigned char* __restrict__ v_cache,
    float* __restrict__ k_scale, float* __restrict__ v_scale,
    const int64_t* __restrict__ slots, int num_tokens, int kv_heads,
    int head_dim, int block_size, int kv_tstride) {
  const int64_t rows = (int64_t)num_tokens * kv_heads;
  const int lane = threadIdx.x & 63;
  for (int64_t row = blockIdx.x * 4 + (threadIdx.x >> 6); row < rows;
       row += (int64_t)gridDim.x * 4) {
    const int g = row % kv_heads;
    const int t = row / kv_heads;
    const int64_t slot = slots[t];
    const int64_t blk = slot / block_size;
    const int off = slot % block_size;
    const bf16_t* src_k = k + (int64_t)t * kv_tstride + g * head_dim;
    const bf16_t* src_v = v + (int64_t)t * kv_tstride + g * head_dim;
    float amax_k = 0.f, amax_v = 0.f;
    for (int d = lane; d < head_dim; d += 64) {
      amax_k = fmaxf(amax_k, fabsf(bf16_to_f32(((const short*)src_k)[d])));
      amax_v = fmaxf(amax_v, fabsf(bf16_to_f32(((const short*)src_v)[d])));
    }
    const float sk = fmaxf(wave_reduce_max(amax_k) * (1.0f / 448.0f), 1e-8f);
    const float sv = fmaxf(wave_reduce_max(amax_v) * (1.0f / 448.0f), 1e-8f);
    const int64_t srow = (blk * kv_heads + g) * block_size + off;
    if (lane == 0) { k_scale[srow] = sk; v_scale[srow] = sv; }
    const float isk = 1.0f / sk, isv = 1.0f / sv;
    unsigned char* dst_k = k_cache + srow * head_dim;
    unsigned char* dst_v = v_cache + srow * head_dim;
    for (int d = lane; d < head_dim; d += 64) {
      dst_k[d] = f32_to_fp8(bf16_to_f32(((const short*)src_k)[d]) * isk);
      dst_v[d] = f32_to_fp8(bf16_to_f32(((const short*)src_v)[d]) * isv);
    }
  }
}

// --------------------------------------------------------------------------
// RoPE and cache store of whole rows in one pass (head size 128): q and k rotated in
// place (entry i with i + 64, as rope_kernel), k and v into the paged cache as bf16, as
// e4m3 with a scale per row (as store_kv_fp8_kernel) or in 4 bits (kv4.h). A thread holds entries c..c+7 and
// c+64..c+71 of a head: 16-byte accesses throughout, where a rotation of 2-byte accesses
// with a workgroup per head and the store behind it took 132 us for 12000 rows of 48
// heads and this takes 50 (320 MB, 6.4 TB/s). held: positions of the cache
// --------------------------------------------------------------------------
template <int KIND>
__global__ void __launch_bounds__(256) rope_store_kernel(
    bf16_t* __restrict__ q, bf16_t* __restrict__ k, const bf16_t* __restrict__ v,
    const int64_t* __restrict__ positions, const float* __restrict__ cos_sin, void* __restrict__ k_cache,
    void* __restrict__ v_cache, void* __restrict__ k_scale, void* __restrict__ v_scale,
    const int64_t* __restrict__ slots, int64_t n, int H, int G, int q_stride, int kv_stride, int block_size, int64_t held) {
  const int heads = H + 2 * G;
  for (int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x; idx < n; idx += (int64_t)gridDim.x * 256) {
    const int piece = (int)(idx & 7);
    const int64_t th = idx >> 3;
    const int64_t t = th / heads;
    const int head = (int)(th - t * heads);
    const bool is_q = head < H, is_v = head >= H + G;
    short* row = is_q ? (short*)q + t * q_stride + head * 128
               : is_v ? (short*)const_cast<bf16_t*>(v) + t * kv_stride + (head - H - G) * 128
                      : (short*)k + t * kv_stride + (head - H) * 128;
    bf16x8_vec a = *reinterpret_cast<const bf16x8_vec*>(row + piece * 8);
    bf16x8_vec b = *reinterpret_cast<const bf16x8_vec*>(row + 64 + piece * 8);
    if (!is_v) {
      const f32x4* cs = reinterpret_cast<const f32x4*>(cos_sin + positions[t] * 128 + piece * 8);
      const f32x4 c[2] = {cs[0], cs[1]}, s[2] = {cs[16], cs[17]};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = bf16_to_f32(a[j]), y = bf16_to_f32(b[j]);
        const float cj = c[j >> 2][j & 3], sj = s[j >> 2][j & 3];
        a[j] = f32_to_bf16(x * cj - y * sj);
        b[j] = f32_to_bf16(y * cj + x * sj);
      }
      *reinterpret_cast<bf16x8_vec*>(row + piece * 8) = a;
      *reinterpret_cast<bf16x8_vec*>(row + 64 + piece * 8) = b;
    }
    if (is_q) continue;
    const int g = head - H - (is_v ? G : 0);
    const int64_t slot = slots[t];
    if (KIND == CACHE_KV4 && (slot < 0 || slot >= held)) continue;       // nobody's, as in kv4_store_kernel; a row's eight lanes as one
    const int64_t at = ((slot / block_size) * G + g) * block_size + slot % block_size;
    if constexpr (KIND == CACHE_KV4) {
      kv4_store_row((uint32_t*)(is_v ? v_cache : k_cache) + at * (KV4_BYTES / 4), (uint32_t*)(is_v ? v_scale : k_scale) + at * KV4_GROUPS,
                    piece, a, b);
    } else if constexpr (KIND == CACHE_FP8) {
      float amax = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        amax = fmaxf(amax, fmaxf(fabsf(bf16_to_f32(a[j])), fabsf(bf16_to_f32(b[j]))));
#pragma unroll
      for (int off = 4; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off));  // the head's eight threads
      const float sc = fmaxf(amax * (1.0f / 448.0f), 1e-8f), inv = 1.0f / sc;
      u8x8_vec lo, hi;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        lo[j] = f32_to_fp8(bf16_to_f32(a[j]) * inv);
        hi[j] = f32_to_fp8(bf16_to_f32(b[j]) * inv);
      }
      unsigned char* o = (unsigned char*)(is_v ? v_cache : k_cache) + at * 128 + piece * 8;
      *reinterpret_cast<u8x8_vec*>(o) = lo;
      *reinterpret_cast<u8x8_vec*>(o + 64) = hi;
      if (piece == 0) ((float*)(is_v ? v_scale : k_scale))[at] = sc;
    } else {
      short* o = (short*)(is_v ? v_cache : k_cache) + at * 128 + piece * 8;
      *reinterpret_cast<bf16x8_vec*>(o) = a;
      *reinterpret_cast<bf16x8_vec*>(o + 64) = b;
    }
  }
}

extern "C" void launch_rope_store(bf16_t* q, bf16_t* k, const bf16_t* v, const int64_t* positions,
                                  const float* cos_sin, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                                  const int64_t* slots, int T, int H, int G, int q_stride, int kv_stride,
                                  int block_size, int64_t held, int kind, hipStream_t stream) {
  const int64_t n = (int64_t)T * (H + 2 * G) * 8;
  const int64_t blocks = (n + 255) / 256;
  const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384));
  hipLaunchKernelGGL(kind == CACHE_KV4   ? rope_store_kernel<CACHE_KV4>
                     : kind == CACHE_FP8 ? rope_store_kernel<CACHE_FP8>
                                         : rope_store_kernel<CACHE_BF16>,
                     grid, dim3(256), 0, stream, q, k, v, positions, cos_sin, k_cache, v_cache, k_scale, v_scale, slots, n, H, G,
                     q_stride, kv_stride, block_size, held);
}
