// The e4m3 linear: y = act(x w^T + bias) of rows and weights held as e4m3 with one
// power-of-two scale for each row and 128 columns of the reduction (fp8.cuh):
//   y[m][n] = sum_b 2^(ex[m][b] + ew[n][b]) sum_{k in b} qx[m][k] qw[n][k] + bias[n].
#include <cuda_runtime.h>
#include <stdint.h>

#include "da3b.h"
#include "fp8.cuh"
#include "fp8.h"
#include "gemm.h"
#include "ops.h"

namespace da3b {

namespace {

__device__ __forceinline__ float fp8_value(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

__device__ __forceinline__ float activate(float v, int act) {
  if (act == kActRelu) return v < 0.f ? 0.f : v;  // NaN stays NaN
  if (act != kActNone) return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
  return v;
}

// Reference form: a CTA computes 32 rows x 128 columns, a thread 2 x 8 of them, from
// dequantised values in shared memory.
__global__ void __launch_bounds__(256) k_linear_fp8(const Fp8Linear a) {
  __shared__ float sx[32][33], sw[32][129];
  const int m0 = blockIdx.y * 32, n0 = blockIdx.x * 128;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int mt = (a.M + 127) / 128, nt = (a.N + 127) / 128;
  float acc[2][8] = {};
  for (int k0 = 0; k0 < a.K; k0 += 32) {
    for (int i = threadIdx.x; i < 32 * 32; i += 256) {
      const int r = i / 32, c = i % 32, m = m0 + r, k = k0 + c;
      sx[c][r] = m < a.M && k < a.K ? fp8_value(a.x[static_cast<size_t>(m) * a.ldx + k]) *
                                          fp8_scale(a.xs[fp8_scale_offset(m, k >> 7, mt)])
                                    : 0.f;
    }
    for (int i = threadIdx.x; i < 128 * 32; i += 256) {
      const int r = i / 32, c = i % 32, n = n0 + r, k = k0 + c;
      sw[c][r] = n < a.N && k < a.K ? fp8_value(a.w[static_cast<size_t>(n) * a.ldw + k]) *
                                          fp8_scale(a.ws[fp8_scale_offset(n, k >> 7, nt)])
                                    : 0.f;
    }
    __syncthreads();
    for (int c = 0; c < 32; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(sx[c][ty * 2 + i], sw[c][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int m = m0 + ty * 2 + i;
    float v[8], amax = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int n = n0 + tx + 16 * j;
      v[j] = n < a.N ? activate(acc[i][j] + (a.bias ? a.bias[n] : 0.f), a.act) : 0.f;
      amax = fmaxf(amax, finite_abs(v[j]));
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (m >= a.M) continue;
    const uint32_t byte = fp8_scale_byte(amax);
    const size_t row = static_cast<size_t>(m) * a.ldo;
    if (a.kind == kFp8OutQ && tx == 0) a.out_scales[fp8_scale_offset(m, n0 >> 7, mt)] = static_cast<uint8_t>(byte);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int n = n0 + tx + 16 * j;
      if (n >= a.N) continue;
      if (a.kind == kFp8OutF16) static_cast<__half*>(a.out)[row + n] = __float2half_rn(v[j]);
      else if (a.kind == kFp8OutBF16) static_cast<__nv_bfloat16*>(a.out)[row + n] = __float2bfloat16_rn(v[j]);
      else if (a.kind == kFp8OutF32) static_cast<float*>(a.out)[row + n] = v[j];
      else if (a.kind == kFp8OutResid) static_cast<float*>(a.out)[row + n] += (a.scale ? a.scale[n] : 1.f) * v[j];
      else static_cast<uint8_t*>(a.out)[row + n] =
          static_cast<uint8_t>(fp8_pack4(fp8_nan_if_inf(v[j]) * fp8_inv_scale(byte), 0.f, 0.f, 0.f) & 255u);
    }
  }
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace

int check_linear_fp8(const Fp8Linear& a) {
  const uintptr_t osz = a.kind == kFp8OutQ ? 1 : (a.kind == kFp8OutF16 || a.kind == kFp8OutBF16) ? 2 : 4;
  if (a.K <= 0 || a.N <= 0 || a.ldx < a.K || a.ldw < a.K || a.ldx % 16 || a.ldw % 16 || a.ldo < a.N ||
      !aligned(a.x, 16) || !aligned(a.w, 16) || !aligned(a.xs, 16) || !aligned(a.ws, 16) || !aligned(a.out, osz) ||
      !aligned(a.bias, 4) || !aligned(a.scale, 4))
    return -1;
  if (a.kind == kFp8OutQ && (a.ldo % 16 || !aligned(a.out, 16) || !aligned(a.out_scales, 16))) return -1;
  return 0;
}

int linear_fp8(const Fp8Linear& a, int* status, cudaStream_t s) {
  if (a.M == 0) return 0;
  const dim3 grid((a.N + 127) / 128, (a.M + 31) / 32);
  (void)status;
  k_linear_fp8<<<grid, 256, 0, s>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

}  // namespace da3b

using namespace da3b;

static int run_linear(const void* x, int M, int K, int ldx, const void* xs, const void* w, int N, int ldw,
                      const void* ws, const float* bias, const float* scale, int act, int kind, void* out, int ldo,
                      void* out_scales, void* stream) {
  if (!x || !xs || !w || !ws || !out || M < 0 || act < 0 || act > 3) return -100;
  const Fp8Linear a = {static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(xs), static_cast<const uint8_t*>(w),
                       static_cast<const uint8_t*>(ws), M, N, K, ldx, ldw, bias, scale, act, kind, out, ldo,
                       static_cast<uint8_t*>(out_scales)};
  if (check_linear_fp8(a)) return -1;
  int* st = device_status_word();
  if (!st) return -101;
  return linear_fp8(a, st, static_cast<cudaStream_t>(stream));
}

extern "C" {

DA3B_API int da3b_linear_fp8(const void* x, int M, int K, int ldx, const void* x_scales, const void* w, int N, int ldw,
                             const void* w_scales, const float* bias, int act, void* out, int out_dtype, int ldo,
                             void* stream) {
  if (out_dtype < kF16 || out_dtype > kF32) return -100;
  return run_linear(x, M, K, ldx, x_scales, w, N, ldw, w_scales, bias, nullptr, act, out_dtype, out, ldo, nullptr,
                    stream);
}

DA3B_API int da3b_linear_fp8_q(const void* x, int M, int K, int ldx, const void* x_scales, const void* w, int N,
                               int ldw, const void* w_scales, const float* bias, int act, void* out_q, int ldo,
                               void* out_scales, void* stream) {
  if (!out_scales) return -100;
  return run_linear(x, M, K, ldx, x_scales, w, N, ldw, w_scales, bias, nullptr, act, kFp8OutQ, out_q, ldo, out_scales,
                    stream);
}

DA3B_API int da3b_linear_fp8_resid_f32(const void* x, int M, int K, int ldx, const void* x_scales, const void* w,
                                       int N, int ldw, const void* w_scales, const float* bias, const float* scale,
                                       float* resid, int ldr, void* stream) {
  return run_linear(x, M, K, ldx, x_scales, w, N, ldw, w_scales, bias, scale, kActNone, kFp8OutResid, resid, ldr,
                    nullptr, stream);
}

}  // extern "C"
