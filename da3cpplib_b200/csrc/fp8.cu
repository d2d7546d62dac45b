// Producers of e4m3 rows with block scales: the quantiser and the LayerNorm that feeds
// a quantised linear.
//
// Both are bounded by memory: each value is read once, and its code and 1/128 of a scale
// byte are written. Eight threads share a block of 128 columns (16 consecutive values
// each), so the block's maximum takes three shuffles, the codes leave as one 16-byte
// store a thread, and 32 threads together hold the four blocks of one scale word.
#include <algorithm>
#include <cuda_runtime.h>
#include <stdint.h>

#include "da3b.h"
#include "fp8.cuh"
#include "fp8.h"

namespace da3b {

namespace {

// 16 consecutive values x[c .. c + 15] of a row as f32, zeros from column K on. VEC: K is
// a multiple of 16 and the row starts on a 16-byte boundary.
template <typename T, bool VEC>
__device__ __forceinline__ void load16(const T* __restrict__ row, int c, int K, float (&v)[16]) {
  if (VEC) {
    if (c < K) {
      const uint4* p = reinterpret_cast<const uint4*>(row + c);
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 u = __ldg(p + i);
          v[4 * i] = __uint_as_float(u.x);
          v[4 * i + 1] = __uint_as_float(u.y);
          v[4 * i + 2] = __uint_as_float(u.z);
          v[4 * i + 3] = __uint_as_float(u.w);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 u = __ldg(p + i);
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            T two[2];
            *reinterpret_cast<uint32_t*>(two) = w[k];
            v[8 * i + 2 * k] = static_cast<float>(two[0]);
            v[8 * i + 2 * k + 1] = static_cast<float>(two[1]);
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = c + i < K ? static_cast<float>(row[c + i]) : 0.f;
  }
}

// Codes and scales of the 512 columns [c0, c0 + 512) of row r that a warp holds, 16 a
// lane (columns c0 + 16 lane ...). Warp-collective.
__device__ __forceinline__ void store_fp8(const float (&v)[16], int r, int c0, int K, int row_tiles,
                                          uint8_t* __restrict__ q, int ldq, uint8_t* __restrict__ scales) {
  const int lane = threadIdx.x & 31;
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) amax = fmaxf(amax, finite_abs(v[i]));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const uint32_t byte = fp8_scale_byte(amax);
  const float inv = fp8_inv_scale(byte);
  float w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = fp8_nan_if_inf(v[i]) * inv;
  const int c = c0 + 16 * lane;
  if (c < K) {  // ldq is a multiple of 16 and at least K
    uint4 u;
    u.x = fp8_pack4(w[0], w[1], w[2], w[3]);
    u.y = fp8_pack4(w[4], w[5], w[6], w[7]);
    u.z = fp8_pack4(w[8], w[9], w[10], w[11]);
    u.w = fp8_pack4(w[12], w[13], w[14], w[15]);
    *reinterpret_cast<uint4*>(q + static_cast<size_t>(r) * ldq + c) = u;
  }
  const uint32_t b0 = __shfl_sync(0xffffffffu, byte, 0), b1 = __shfl_sync(0xffffffffu, byte, 8);
  const uint32_t b2 = __shfl_sync(0xffffffffu, byte, 16), b3 = __shfl_sync(0xffffffffu, byte, 24);
  if (lane == 0)
    *reinterpret_cast<uint32_t*>(scales + fp8_scale_offset(r, c0 >> 7, row_tiles)) =
        b0 | (b1 << 8) | (b2 << 16) | (b3 << 24);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    k_quantize_fp8(const T* __restrict__ x, int rows, int K, int ldx, uint8_t* __restrict__ q, int ldq,
                   uint8_t* __restrict__ scales) {
  const int groups = (K + 511) / 512, row_tiles = (rows + 127) / 128;
  const long items = static_cast<long>(rows) * groups;
  const long step = static_cast<long>(gridDim.x) * 8;
  for (long it = static_cast<long>(blockIdx.x) * 8 + (threadIdx.x >> 5); it < items; it += step) {
    const int r = static_cast<int>(it / groups), c0 = static_cast<int>(it % groups) * 512;
    float v[16];
    load16<T, VEC>(x + static_cast<size_t>(r) * ldx, c0 + 16 * (threadIdx.x & 31), K, v);
    store_fp8(v, r, c0, K, row_tiles, q, ldq, scales);
  }
}

// LayerNorm of f32 rows, two-pass mean and variance in f32 over the row held in
// registers, quantised. WARPS warps share a row, each with up to NV groups of 512
// columns; rows of at most 2048 columns take one warp, longer ones eight.
template <int WARPS, int NV, bool VEC>
__global__ void __launch_bounds__(256)
    k_layernorm_fp8(const float* __restrict__ x, int rows, int K, int ldx, const float* __restrict__ g,
                    const float* __restrict__ b, float eps, uint8_t* __restrict__ q, int ldq,
                    uint8_t* __restrict__ scales) {
  __shared__ float part[2][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = WARPS == 1 ? blockIdx.x * 8 + warp : blockIdx.x;
  if (WARPS == 1 && r >= rows) return;
  const int sub = WARPS == 1 ? 0 : warp;
  const float* row = x + static_cast<size_t>(r) * ldx;
  float v[NV][16];
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    load16<float, VEC>(row, (j * WARPS + sub) * 512 + 16 * lane, K, v[j]);
#pragma unroll
    for (int i = 0; i < 16; ++i) s += v[j][i];
  }
  auto row_sum = [&](float t, int which) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (WARPS == 1) return t;
    if (lane == 0) part[which][warp] = t;
    __syncthreads();
    float u = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) u += part[which][i];
    return u;
  };
  const float mean = row_sum(s, 0) / K;
  float d2 = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float d = v[j][i] - mean;
      if ((j * WARPS + sub) * 512 + 16 * lane + i < K) d2 = fmaf(d, d, d2);
    }
  const float rstd = 1.0f / sqrtf(row_sum(d2, 1) / K + eps);
  const int row_tiles = (rows + 127) / 128;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c0 = (j * WARPS + sub) * 512, c = c0 + 16 * lane;
    if (c0 >= K) break;  // the whole warp
    float y[16];
    if (VEC) {
      float gg[16], bb[16];
      load16<float, true>(g, c, K, gg);
      if (b) load16<float, true>(b, c, K, bb);
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = c < K ? (v[j][i] - mean) * rstd * gg[i] + (b ? bb[i] : 0.f) : 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        y[i] = c + i < K ? (v[j][i] - mean) * rstd * __ldg(g + c + i) + (b ? __ldg(b + c + i) : 0.f) : 0.f;
    }
    store_fp8(y, r, c0, K, row_tiles, q, ldq, scales);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool bad_codes(const uint8_t* q, int ldq, const uint8_t* scales, int K) {
  return ldq < K || ldq % 16 || !aligned16(q) || !aligned16(scales);
}

template <typename T>
int launch_quantize(const void* xv, int rows, int K, int ldx, uint8_t* q, int ldq, uint8_t* scales, cudaStream_t s) {
  const T* x = static_cast<const T*>(xv);
  if (reinterpret_cast<uintptr_t>(x) % sizeof(T)) return -1;
  const long items = static_cast<long>(rows) * ((K + 511) / 512);
  const unsigned blocks = static_cast<unsigned>(std::min<long>((items + 7) / 8, 148L * 64));
  if (K % 16 == 0 && (static_cast<size_t>(ldx) * sizeof(T)) % 16 == 0 && aligned16(x))
    k_quantize_fp8<T, true><<<blocks, 256, 0, s>>>(x, rows, K, ldx, q, ldq, scales);
  else
    k_quantize_fp8<T, false><<<blocks, 256, 0, s>>>(x, rows, K, ldx, q, ldq, scales);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

}  // namespace

int quantize_fp8(const void* x, int dtype, int rows, int K, int ldx, uint8_t* q, int ldq, uint8_t* scales,
                 cudaStream_t s) {
  if (K <= 0 || ldx < K || bad_codes(q, ldq, scales, K)) return -1;
  if (rows == 0) return 0;
  switch (dtype) {
    case kF16: return launch_quantize<__half>(x, rows, K, ldx, q, ldq, scales, s);
    case kBF16: return launch_quantize<__nv_bfloat16>(x, rows, K, ldx, q, ldq, scales, s);
    case kF32: return launch_quantize<float>(x, rows, K, ldx, q, ldq, scales, s);
  }
  return -1;
}

int layernorm_fp8(const float* x, int rows, int K, int ldx, const float* g, const float* b, float eps, uint8_t* q,
                  int ldq, uint8_t* scales, cudaStream_t s) {
  if (K <= 0 || K > 16384 || ldx < K || bad_codes(q, ldq, scales, K) || !(eps >= 0.f)) return -1;
  if (reinterpret_cast<uintptr_t>(x) % 4 || reinterpret_cast<uintptr_t>(g) % 4 || reinterpret_cast<uintptr_t>(b) % 4)
    return -1;
  if (rows == 0) return 0;
  const bool vec = K % 16 == 0 && ldx % 4 == 0 && aligned16(x) && aligned16(g) && aligned16(b);
  const unsigned per_warp = static_cast<unsigned>((rows + 7) / 8), per_block = static_cast<unsigned>(rows);
#define DA3B_LNF8(W, NV, GRID)                                                                          \
  do {                                                                                                  \
    if (vec) k_layernorm_fp8<W, NV, true><<<GRID, 256, 0, s>>>(x, rows, K, ldx, g, b, eps, q, ldq, scales); \
    else k_layernorm_fp8<W, NV, false><<<GRID, 256, 0, s>>>(x, rows, K, ldx, g, b, eps, q, ldq, scales);    \
  } while (0)
  if (K <= 512) DA3B_LNF8(1, 1, per_warp);
  else if (K <= 1024) DA3B_LNF8(1, 2, per_warp);
  else if (K <= 2048) DA3B_LNF8(1, 4, per_warp);
  else if (K <= 8192) DA3B_LNF8(8, 2, per_block);
  else DA3B_LNF8(8, 4, per_block);
#undef DA3B_LNF8
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

}  // namespace da3b

using namespace da3b;

extern "C" {

DA3B_API size_t da3b_fp8_scale_bytes(int rows, int K) { return rows > 0 && K > 0 ? fp8_scale_bytes(rows, K) : 0; }

DA3B_API int da3b_quantize_fp8(const void* x, int dtype, int rows, int K, int ldx, void* q, int ldq, void* scales,
                               void* stream) {
  if (!x || !q || !scales || rows < 0) return -100;
  return quantize_fp8(x, dtype, rows, K, ldx, static_cast<uint8_t*>(q), ldq, static_cast<uint8_t*>(scales),
                      static_cast<cudaStream_t>(stream));
}

DA3B_API int da3b_layernorm_fp8(const float* x, int rows, int K, int ldx, const float* gamma, const float* beta,
                                float eps, void* q, int ldq, void* scales, void* stream) {
  if (!x || !gamma || !q || !scales || rows < 0) return -100;
  return layernorm_fp8(x, rows, K, ldx, gamma, beta, eps, static_cast<uint8_t*>(q), ldq,
                       static_cast<uint8_t*>(scales), static_cast<cudaStream_t>(stream));
}

}  // extern "C"
