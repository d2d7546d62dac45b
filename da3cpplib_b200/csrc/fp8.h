// Launchers of the 8-bit floating-point path (fp8.cu, fp8_linear.cu).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace da3b {

// Element types of the kernel-level ABI's typed arguments.
enum DType : int { kF16 = 0, kBF16 = 1, kF32 = 2 };

// Bytes of the scale tiles of a [rows][K] matrix: 512 for each 128 rows x 512 columns.
inline size_t fp8_scale_bytes(int rows, int K) {
  return (static_cast<size_t>(K) + 511) / 512 * ((static_cast<size_t>(rows) + 127) / 128) * 512;
}

int quantize_fp8(const void* x, int dtype, int rows, int K, int ldx, uint8_t* q, int ldq, uint8_t* scales,
                 cudaStream_t s);
int layernorm_fp8(const float* x, int rows, int K, int ldx, const float* g, const float* b, float eps, uint8_t* q,
                  int ldq, uint8_t* scales, cudaStream_t s);

// Output of the e4m3 linear.
enum Fp8Out : int { kFp8OutF16 = 0, kFp8OutBF16 = 1, kFp8OutF32 = 2, kFp8OutResid = 3, kFp8OutQ = 4 };

struct Fp8Linear {
  const uint8_t* x;   // [M][ldx] e4m3
  const uint8_t* xs;  // scale tiles
  const uint8_t* w;   // [N][ldw] e4m3
  const uint8_t* ws;
  int M, N, K, ldx, ldw;
  const float* bias;   // [N] or null
  const float* scale;  // [N] or null (kFp8OutResid)
  int act;             // Act (gemm.h)
  int kind;            // Fp8Out
  void* out;           // [M][ldo] of the output type; f32 residual; or e4m3 codes
  int ldo;
  uint8_t* out_scales;  // kFp8OutQ
};

// 0, or -1 where sizes, leading dimensions or alignments are not served (no GPU work).
int check_linear_fp8(const Fp8Linear& a);
int linear_fp8(const Fp8Linear& a, int* status, cudaStream_t s);

}  // namespace da3b
