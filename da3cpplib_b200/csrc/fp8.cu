// Producers of e4m3 rows with block scales: the quantiser and the LayerNorm that feeds
// a quantised linear.
//
// Both are bounded by memory: each value is read once, and its code and 1/128 of a scale
// byte are written. Eight threads share a block of 128 columns (16 consecutive values
// each), so the block's maximum takes three shuffles, the codes leave as one 16-byte
// store a thread, and 32 threads together hold the four blocks of one scale word.
#include <algorithm>
#include <atomic>
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "da3b.h"
#include "fp8.cuh"
#include "fp8.h"
#include "launch.h"
#include "ptx.cuh"

namespace da3b {

namespace {

// 16 consecutive values x[c .. c + 15] of a row as f32, zeros from column K on. VEC: K is
// a multiple of 16 and the row starts on a 32-byte boundary. Plain loads, not those of the
// read-only path (nor of pointers that the compiler may take for it): a kernel that starts
// while the one ahead of it is still running may be reading what that one writes.
template <typename T, bool VEC>
__device__ __forceinline__ void load16(const T* row, int c, int K, float (&v)[16]) {
  if (VEC) {
    if (c < K) {
      // 32 bytes a load: a warp's loads cover 1024 consecutive bytes
      uint32_t w[sizeof(T) * 4];
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w[8 * i]), "=r"(w[8 * i + 1]), "=r"(w[8 * i + 2]), "=r"(w[8 * i + 3]), "=r"(w[8 * i + 4]),
                       "=r"(w[8 * i + 5]), "=r"(w[8 * i + 6]), "=r"(w[8 * i + 7])
                     : "l"(reinterpret_cast<const uint32_t*>(row + c) + 8 * i));
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(w[i]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          T two[2];
          *reinterpret_cast<uint32_t*>(two) = w[k];
          v[2 * k] = static_cast<float>(two[0]);
          v[2 * k + 1] = static_cast<float>(two[1]);
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
// lane (columns c0 + 16 lane ...); the scale bytes of the row's blocks from c0 on.
// Warp-collective. The kernels here are bounded by instructions as much as by memory, so
// the maximum is taken without looking at infinities (NaN drops out of it by itself) and
// only a warp that meets one does it again.
__device__ __forceinline__ void store_fp8(float (&v)[16], int r, int c0, int K, uint8_t* __restrict__ q, int ldq,
                                          uint8_t* __restrict__ scale4) {
  const int lane = threadIdx.x & 31;
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(v[i]));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (__any_sync(0xffffffffu, amax > kFltMax)) {
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      amax = fmaxf(amax, finite_abs(v[i]));
      v[i] = fp8_nan_if_inf(v[i]);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  }
  const uint32_t byte = fp8_scale_byte(amax);
  const float inv = fp8_inv_scale(byte);
  const int c = c0 + 16 * lane;
  if (c < K) {  // ldq is a multiple of 16 and at least K
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 s2 = make_float2(inv, inv);
      const float2 a = __fmul2_rn(make_float2(v[4 * i], v[4 * i + 1]), s2);
      const float2 b = __fmul2_rn(make_float2(v[4 * i + 2], v[4 * i + 3]), s2);
      w[i] = fp8_pack4(a.x, a.y, b.x, b.y);
    }
    *reinterpret_cast<uint4*>(q + static_cast<size_t>(r) * ldq + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if ((lane & 7) == 0) scale4[lane >> 3] = static_cast<uint8_t>(byte);
}

// A warp takes one row and up to two groups of 512 columns of it (blockIdx.y), both loaded
// before either is worked on. f16 rows, 87680 x 1024: 49 us, 5.5 TB/s (0.84 of a copy); the
// warps wait for their loads, with 4 KB in flight each and 31 of them an SM.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    k_quantize_fp8(const T* x, int rows, int K, int ldx, uint8_t* __restrict__ q, int ldq,
                   uint8_t* __restrict__ scales) {
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5);
  pdl_trigger();
  if (r >= rows) return;
  pdl_wait();
  const int row_tiles = (rows + 127) / 128, c0 = blockIdx.y * 1024, lane = threadIdx.x & 31;
  const T* row = x + static_cast<size_t>(r) * ldx;
  float v[16], w[16];
  load16<T, VEC>(row, c0 + 16 * lane, K, v);
  const bool two = c0 + 512 < K;
  if (two) load16<T, VEC>(row, c0 + 512 + 16 * lane, K, w);
  uint8_t* s4 = scales + fp8_scale_offset(r, c0 >> 7, row_tiles);
  store_fp8(v, r, c0, K, q, ldq, s4);
  if (two) store_fp8(w, r, c0 + 512, K, q, ldq, s4 + static_cast<size_t>(row_tiles) * 512);
}

// LayerNorm of f32 rows, two-pass mean and variance in f32 over the row held in
// registers, quantised. WARPS warps share a row, each with up to NV groups of 512
// columns; rows of at most 2048 columns take one warp, longer ones eight.
template <int WARPS, int NV, bool VEC>
__global__ void __launch_bounds__(256)
    k_layernorm_fp8(const float* x, int rows, int K, int ldx, const float* g,
                    const float* b, float eps, uint8_t* __restrict__ q, int ldq,
                    uint8_t* __restrict__ scales) {
  __shared__ float part[2][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = WARPS == 1 ? blockIdx.x * 8 + warp : blockIdx.x;
  pdl_trigger();
  if (WARPS == 1 && r >= rows) return;
  pdl_wait();
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
        y[i] = c + i < K ? (v[j][i] - mean) * rstd * g[c + i] + (b ? b[c + i] : 0.f) : 0.f;
    }
    store_fp8(y, r, c0, K, q, ldq, scales + fp8_scale_offset(r, c0 >> 7, row_tiles));
  }
}

// The same for rows of up to 1024 columns that load16 reads 32 bytes at a time. A warp walks
// over its rows, loads the next one before it works on the one it holds, and keeps gamma and
// beta in registers: read again for each row they were two thirds of what passed through L1,
// whose 74 % was the busiest of the form above (87680 x 1024: 97 us, here 78 us or 5.8 TB/s,
// 0.88 of a copy; walking without the registers 91 us). Rows of 768 columns leave a quarter
// of the lanes without work: 4.6 TB/s.
template <int NV>
constexpr int kWalkBlocks = NV == 1 ? 5 : 3;  // resident on an SM, by registers

template <int NV>
__global__ void __launch_bounds__(128, kWalkBlocks<NV>)
    k_layernorm_fp8_walk(const float* x, int rows, int K, int ldx, const float* g,
                         const float* b, float eps, uint8_t* __restrict__ q, int ldq,
                         uint8_t* __restrict__ scales) {
  const int lane = threadIdx.x & 31, step = gridDim.x * 4;
  const int row_tiles = (rows + 127) / 128;
  int r = blockIdx.x * 4 + (threadIdx.x >> 5);
  pdl_trigger();
  if (r >= rows) return;
  pdl_wait();
  float v[NV][16], n[NV][16];
#pragma unroll
  for (int j = 0; j < NV; ++j) load16<float, true>(x + static_cast<size_t>(r) * ldx, j * 512 + 16 * lane, K, n[j]);
  float gg[NV][16], bb[NV][16];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    load16<float, true>(g, j * 512 + 16 * lane, K, gg[j]);
#pragma unroll
    for (int i = 0; i < 16; ++i) bb[j][i] = 0.f;
    if (b) load16<float, true>(b, j * 512 + 16 * lane, K, bb[j]);
  }
  while (true) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) v[j][i] = n[j][i];
    const bool more = r < rows - step;
    if (more) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        load16<float, true>(x + static_cast<size_t>(r + step) * ldx, j * 512 + 16 * lane, K, n[j]);
    }
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) s += v[j][i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float mean = s / K;
    float d2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool in = j * 512 + 16 * lane < K;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        v[j][i] -= mean;
        d2 = in ? fmaf(v[j][i], v[j][i], d2) : d2;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d2 += __shfl_xor_sync(0xffffffffu, d2, o);
    const float rstd = 1.0f / sqrtf(d2 / K + eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c0 = j * 512;
      if (c0 >= K) break;  // the whole warp
#pragma unroll
      for (int i = 0; i < 16; ++i) v[j][i] = v[j][i] * rstd * gg[j][i] + bb[j][i];
      store_fp8(v[j], r, c0, K, q, ldq, scales + fp8_scale_offset(r, c0 >> 7, row_tiles));
    }
    if (!more) break;
    r += step;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; }

bool bad_codes(const uint8_t* q, int ldq, const uint8_t* scales, int K) {
  return ldq < K || ldq % 16 || !aligned16(q) || !aligned16(scales);
}

template <typename T>
int launch_quantize(const void* xv, int rows, int K, int ldx, uint8_t* q, int ldq, uint8_t* scales, cudaStream_t s) {
  const T* x = static_cast<const T*>(xv);
  const dim3 grid((static_cast<unsigned>(rows) + 7) / 8, (static_cast<unsigned>(K) + 1023) / 1024);
  if (grid.y > 65535) return -1;
  cudaError_t e;
  if (K % 16 == 0 && (static_cast<size_t>(ldx) * sizeof(T)) % 32 == 0 && aligned32(x))
    e = launch_pdl(k_quantize_fp8<T, true>, grid, 256, 0, s, 1, x, rows, K, ldx, q, ldq, scales);
  else
    e = launch_pdl(k_quantize_fp8<T, false>, grid, 256, 0, s, 1, x, rows, K, ldx, q, ldq, scales);
  return e == cudaSuccess ? 0 : -4;
}

}  // namespace

bool usable_here(std::initializer_list<const void*> buffers) {
  typedef CUresult (*PFN_pointerAttribute)(void*, CUpointer_attribute, CUdeviceptr);
  static std::atomic<PFN_pointerAttribute> known{nullptr};
  PFN_pointerAttribute ask = known.load(std::memory_order_acquire);
  if (!ask) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuPointerGetAttribute", &f, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      return false;
    ask = reinterpret_cast<PFN_pointerAttribute>(f);
    known.store(ask, std::memory_order_release);
  }
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  for (const void* p : buffers) {
    if (!p) continue;
    const CUdeviceptr d = reinterpret_cast<CUdeviceptr>(p);
    int at = -1;
    if (ask(&at, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL, d) != CUDA_SUCCESS) return false;
    if (at == dev) continue;
    // pinned and managed memory belong to no device in particular (the one named is that which
    // was current when they were allocated)
    unsigned type = 0, managed = 0;
    if (ask(&type, CU_POINTER_ATTRIBUTE_MEMORY_TYPE, d) == CUDA_SUCCESS && type == CU_MEMORYTYPE_HOST) continue;
    if (ask(&managed, CU_POINTER_ATTRIBUTE_IS_MANAGED, d) != CUDA_SUCCESS || !managed) return false;
  }
  return true;
}

int sm_count(int dev) {
  static std::atomic<int> counts[64];
  int n = counts[dev & 63].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    counts[dev & 63].store(n, std::memory_order_relaxed);
  }
  return n;
}

int quantize_fp8(const void* x, int dtype, int rows, int K, int ldx, uint8_t* q, int ldq, uint8_t* scales,
                 cudaStream_t s) {
  if (K <= 0 || K > kMostCount || rows > kMostCount || ldx < K || bad_codes(q, ldq, scales, K) || dtype < kF16 ||
      dtype > kF32 || reinterpret_cast<uintptr_t>(x) % (dtype == kF32 ? 4 : 2))
    return -1;
  if (rows == 0) return 0;
  if (!usable_here({x, q, scales})) return -104;
  switch (dtype) {
    case kF16: return launch_quantize<__half>(x, rows, K, ldx, q, ldq, scales, s);
    case kBF16: return launch_quantize<__nv_bfloat16>(x, rows, K, ldx, q, ldq, scales, s);
    case kF32: return launch_quantize<float>(x, rows, K, ldx, q, ldq, scales, s);
  }
  return -1;
}

int layernorm_fp8(const float* x, int rows, int K, int ldx, const float* g, const float* b, float eps, uint8_t* q,
                  int ldq, uint8_t* scales, cudaStream_t s) {
  if (K <= 0 || K > 16384 || rows > kMostCount || ldx < K || bad_codes(q, ldq, scales, K) || !(eps >= 0.f)) return -1;
  if (reinterpret_cast<uintptr_t>(x) % 4 || reinterpret_cast<uintptr_t>(g) % 4 || reinterpret_cast<uintptr_t>(b) % 4)
    return -1;
  if (rows == 0) return 0;
  if (!usable_here({x, g, b, q, scales})) return -104;
  const bool vec = K % 16 == 0 && ldx % 8 == 0 && aligned32(x) && aligned32(g) && aligned32(b);
  const unsigned per_warp = static_cast<unsigned>((rows + 7) / 8), per_block = static_cast<unsigned>(rows);
  cudaError_t e;
#define DA3B_LNF8(W, NV, GRID)                                                                                        \
  do {                                                                                                                \
    if (vec) e = launch_pdl(k_layernorm_fp8<W, NV, true>, dim3(GRID), 256, 0, s, 1, x, rows, K, ldx, g, b, eps, q,    \
                            ldq, scales);                                                                             \
    else e = launch_pdl(k_layernorm_fp8<W, NV, false>, dim3(GRID), 256, 0, s, 1, x, rows, K, ldx, g, b, eps, q, ldq,  \
                        scales);                                                                                      \
  } while (0)
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned walk = static_cast<unsigned>(sm_count(dev) * (K <= 512 ? kWalkBlocks<1> : kWalkBlocks<2>));
  const dim3 walkers(std::min((static_cast<unsigned>(rows) + 3) / 4, walk));
  if (vec && K <= 512)
    e = launch_pdl(k_layernorm_fp8_walk<1>, walkers, 128, 0, s, 1, x, rows, K, ldx, g, b, eps, q, ldq, scales);
  else if (vec && K <= 1024)
    e = launch_pdl(k_layernorm_fp8_walk<2>, walkers, 128, 0, s, 1, x, rows, K, ldx, g, b, eps, q, ldq, scales);
  else if (K <= 512) DA3B_LNF8(1, 1, per_warp);
  else if (K <= 1024) DA3B_LNF8(1, 2, per_warp);
  else if (K <= 2048) DA3B_LNF8(1, 4, per_warp);
  else if (K <= 8192) DA3B_LNF8(8, 2, per_block);
  else DA3B_LNF8(8, 4, per_block);
#undef DA3B_LNF8
  return e == cudaSuccess ? 0 : -4;
}

}  // namespace da3b

using namespace da3b;

extern "C" {

DA3B_API size_t da3b_fp8_scale_bytes(int rows, int K) { return rows > 0 && K > 0 ? fp8_scale_bytes(rows, K) : 0; }

DA3B_API int da3b_quantize_fp8(const void* x, int dtype, int rows, int K, int ldx, void* q, int ldq, void* scales,
                               void* stream) {
  if (rows < 0 || (rows > 0 && (!x || !q || !scales))) return -100;
  return quantize_fp8(x, dtype, rows, K, ldx, static_cast<uint8_t*>(q), ldq, static_cast<uint8_t*>(scales),
                      static_cast<cudaStream_t>(stream));
}

DA3B_API int da3b_layernorm_fp8(const float* x, int rows, int K, int ldx, const float* gamma, const float* beta,
                                float eps, void* q, int ldq, void* scales, void* stream) {
  if (!gamma || rows < 0 || (rows > 0 && (!x || !q || !scales))) return -100;
  return layernorm_fp8(x, rows, K, ldx, gamma, beta, eps, static_cast<uint8_t*>(q), ldq,
                       static_cast<uint8_t*>(scales), static_cast<cudaStream_t>(stream));
}

}  // extern "C"
