// Activations of the linears' epilogues.
#pragma once
#include <cuda_fp16.h>

#include "gemm.h"
#include "ptx.cuh"

namespace da3b {

// erf(z) by Abramowitz & Stegun, Handbook of Mathematical Functions, formula 7.1.26:
// erf(z) = 1 - (a1 t + a2 t^2 + a3 t^3 + a4 t^4 + a5 t^5) e^(-z^2), t = 1 / (1 + p z),
// z >= 0, |error| <= 1.5e-7 (odd extension for z < 0). Far below the f16 rounding of
// the GELU output it feeds.
__device__ __forceinline__ float erf_as(float z) {
  const float az = fabsf(z);
  const float t = __fdividef(1.0f, fmaf(0.3275911f, az, 1.0f));
  float y = fmaf(1.061405429f, t, -1.453152027f);
  y = fmaf(y, t, 1.421413741f);
  y = fmaf(y, t, -0.284496736f);
  y = fmaf(y, t, 0.254829592f);
  y *= t;
  const float e = ex2_approx(-az * az * 1.4426950408889634f);
  return copysignf(fmaf(-y, e, 1.0f), z);
}
// Exact-form GELU 0.5 x (1 + erf(x / sqrt 2)) (ggml_gelu_erf, src/ggml_extend.hpp:22-25).
__device__ __forceinline__ float gelu_erf(float v) { return 0.5f * v * (1.0f + erf_as(v * 0.70710678118654752f)); }

// gelu_erf of two values with packed f32x2 arithmetic (sm_100): the same operations in
// the same order as gelu_erf, so each result is bit-identical to the scalar one, in
// about half the instructions.
__device__ __forceinline__ float2 f2c(float c) { return make_float2(c, c); }
__device__ __forceinline__ float2 gelu_erf2(float2 v) {
  const float2 z = __fmul2_rn(v, f2c(0.70710678118654752f));
  const float2 az = make_float2(fabsf(z.x), fabsf(z.y));
  const float2 d = __ffma2_rn(f2c(0.3275911f), az, f2c(1.0f));
  const float2 t = make_float2(__fdividef(1.0f, d.x), __fdividef(1.0f, d.y));
  float2 y = __ffma2_rn(f2c(1.061405429f), t, f2c(-1.453152027f));
  y = __ffma2_rn(y, t, f2c(1.421413741f));
  y = __ffma2_rn(y, t, f2c(-0.284496736f));
  y = __ffma2_rn(y, t, f2c(0.254829592f));
  y = __fmul2_rn(y, t);
  const float2 w = __fmul2_rn(__fmul2_rn(make_float2(-az.x, -az.y), az), f2c(1.4426950408889634f));
  const float2 ex = make_float2(ex2_approx(w.x), ex2_approx(w.y));
  float2 r = __ffma2_rn(make_float2(-y.x, -y.y), ex, f2c(1.0f));
  r = make_float2(copysignf(r.x, z.x), copysignf(r.y, z.y));
  return __fmul2_rn(__fmul2_rn(f2c(0.5f), v), __fadd2_rn(f2c(1.0f), r));
}

// Exact-form GELU with erf from Abramowitz & Stegun formula 7.1.28:
// erf(z) = 1 - (1 + a1 z + a2 z^2 + ... + a6 z^6)^-16, z >= 0, |error| <= 3e-7. With
// r = (1 + ...)^-16, 1 + erf(x / sqrt 2) is 2 - r for x >= 0 and r for x < 0 (no
// cancellation for negative x); one reciprocal (MUFU) and no exponential per value.
__device__ __forceinline__ float gelu_r(float v) {
  const float z = fabsf(v * 0.70710678118654752f);
  float p = fmaf(0.0000430638f, z, 0.0002765672f);
  p = fmaf(p, z, 0.0001520143f);
  p = fmaf(p, z, 0.0092705272f);
  p = fmaf(p, z, 0.0422820123f);
  p = fmaf(p, z, 0.0705230784f);
  p = fmaf(p, z, 1.0f);
  float r = __fdividef(1.0f, p);
  r *= r;
  r *= r;
  r *= r;
  r *= r;
  return 0.5f * v * (v >= 0.0f ? 2.0f - r : r);
}
// gelu_r of two values with packed f32x2 arithmetic, the same operations in the same
// order (bit-identical to the scalar form).
__device__ __forceinline__ float2 gelu_r2(float2 v) {
  const float2 zz = __fmul2_rn(v, f2c(0.70710678118654752f));
  const float2 z = make_float2(fabsf(zz.x), fabsf(zz.y));
  float2 p = __ffma2_rn(f2c(0.0000430638f), z, f2c(0.0002765672f));
  p = __ffma2_rn(p, z, f2c(0.0001520143f));
  p = __ffma2_rn(p, z, f2c(0.0092705272f));
  p = __ffma2_rn(p, z, f2c(0.0422820123f));
  p = __ffma2_rn(p, z, f2c(0.0705230784f));
  p = __ffma2_rn(p, z, f2c(1.0f));
  float2 r = make_float2(__fdividef(1.0f, p.x), __fdividef(1.0f, p.y));
  r = __fmul2_rn(r, r);
  r = __fmul2_rn(r, r);
  r = __fmul2_rn(r, r);
  r = __fmul2_rn(r, r);
  const float2 t = make_float2(v.x >= 0.0f ? 2.0f - r.x : r.x, v.y >= 0.0f ? 2.0f - r.y : r.y);
  return __fmul2_rn(__fmul2_rn(f2c(0.5f), v), t);
}

__device__ __forceinline__ float apply_act(float v, int act) {
  if (act == kActRelu) return fmaxf(v, 0.0f);
  if (act == kActGelu) return gelu_erf(v);
  if (act == kActGeluR) return gelu_r(v);
  return v;
}

}  // namespace da3b
