// Epilogue arithmetic of the gated and 8-bit products, in FP32; each output is
// rounded to FP16 once, by the caller.
#pragma once

#include "common.cuh"

namespace ctb {

enum : int { kSilu = 0, kGelu = 1 };

// g / (1 + exp(-g)); the denominator overflows to infinity below -88, where
// the result is -0 to FP32's precision.
__device__ __forceinline__ float silu(float g) { return g / (1.0f + __expf(-g)); }

__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// exp(x) as 2^(x log2 e), 2^-21 relative for the exponents that matter; results
// below the normal range are 0.
__device__ __forceinline__ float exp_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}

// The activations of the tensor-core epilogues, in the fewest instructions
// (one reciprocal for two gates took fewer special functions and was 2 %
// slower). silu_fast is -0 where exp(-g) overflows.
__device__ __forceinline__ float silu_fast(float g) { return g * reciprocal(1.0f + exp_fast(-g)); }

// erf-GELU by the formula of erf_as7126.
__device__ __forceinline__ float gelu_fast(float g) {
  const float z = fabsf(g) * 0.7071067811865476f;
  const float t = reciprocal(fmaf(0.3275911f, z, 1.0f));
  float poly = fmaf(1.061405429f, t, -1.453152027f);
  poly = fmaf(poly, t, 1.421413741f);
  poly = fmaf(poly, t, -0.284496736f);
  poly = fmaf(poly, t, 0.254829592f);
  const float erf = fmaf(-poly * t, exp_fast(-z * z), 1.0f);
  return 0.5f * g * (1.0f + copysignf(erf, g));
}

__device__ __forceinline__ float gated(float gate, float up, int activation) {
  return (activation == kSilu ? silu(gate) : gelu_erf(gate)) * up;
}

// acc is the exact sum of 8-bit products; FP32 keeps 24 of its bits, more
// than the FP16 result. The scales are multiplied first: their product is the
// same for every kernel form, so all forms round alike.
__device__ __forceinline__ float dequantized(int acc, float row_scale, float column_scale, float bias) {
  return fmaf(static_cast<float>(acc), row_scale * column_scale, bias);
}

}  // namespace ctb
