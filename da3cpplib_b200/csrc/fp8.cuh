// e4m3 with one power-of-two scale for each row and 128 columns: device helpers.
//
// A block of 128 values x is held as codes q (e4m3) and a byte s = e + 127 with
// x ~ q * 2^e; e is the smallest integer with max|x| <= 448 * 2^e (448 = 1.75 * 2^8, the
// largest e4m3 value), at least -127, and 0 for a block of zeros. Scaling by a power of
// two is exact, so the only rounding is the one to e4m3 (3 mantissa bits: half a step is
// 2^-4 of the value, or 2^-10 * 2^e below 2^-6 * 2^e), the codes do not depend on how
// they are computed, and the tensor cores apply the scales themselves (ue8m0 bytes).
// e4m3 has no infinity: infinities and NaN both become NaN, and the scale is that of the
// block's finite values.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace da3b {

constexpr float kFltMax = 3.402823466e38f;

// |v| for the block maximum: 0 for infinities and NaN.
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= kFltMax ? a : 0.f;
}

// Scale byte e + 127 of a block whose largest finite |x| is amax: adding 0x1fffff to the
// float's bits carries into the exponent exactly when its mantissa is above 1.75, and
// 448 = 1.75 * 2^8. Subnormal amax clamps to e = -127.
__device__ __forceinline__ uint32_t fp8_scale_byte(float amax) {
  if (amax == 0.f) return 127u;
  const int e = static_cast<int>((__float_as_uint(amax) + 0x1fffffu) >> 23) - 8;
  return static_cast<uint32_t>(max(e, 0));
}

// 2^-(byte - 127); byte <= 247 for finite f32 data (amax < 2^128), so -e >= -120.
__device__ __forceinline__ float fp8_inv_scale(uint32_t byte) {
  return __uint_as_float((254u - byte) << 23);  // byte 0: 2^127
}

// 2^(byte - 127)
__device__ __forceinline__ float fp8_scale(uint32_t byte) {
  return byte == 0 ? 5.877471754e-39f : __uint_as_float(byte << 23);
}

__device__ __forceinline__ float fp8_nan_if_inf(float v) {
  return fabsf(v) <= kFltMax ? v : __uint_as_float(0x7fffffffu);
}

// Codes of four scaled values, first in the low byte.
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// Offset of the scale byte of (row r, block b) in the scale tiles of a matrix of
// row_tiles x 128 rows: tiles [K/512][row tile] of [32][4][4] bytes, row 32 c + l of the
// tile and block 4 g + j at [l][c][j], the order in which tcgen05.cp lays 128 rows of four
// blocks out in tensor memory (lane l, column c, byte j).
__device__ __forceinline__ size_t fp8_scale_offset(int r, int b, int row_tiles) {
  const size_t tile = static_cast<size_t>(b >> 2) * row_tiles + (r >> 7);
  return tile * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (b & 3);
}

}  // namespace da3b
