// Epilogue arithmetic of the gated and 8-bit products, in FP32; each output is
// rounded to FP16 once, by the caller.
#pragma once

#include "common.cuh"

namespace ctb {

enum : int { kSilu = 0, kGelu = 1 };

__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// exp(x) as 2^(x log2 e). The product's rounding and the constant's move the
// exponent by up to |x| log2(e) 2^-23, so the result is right to |x| 2^-23 of
// itself, and 2^-22 more for ex2.approx; results below the normal range are 0.
__device__ __forceinline__ float exp_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}

// g / (1 + exp(-g)) in the fewest instructions (one reciprocal for two gates
// took fewer special functions and was 2 % slower); -0 where exp(-g)
// overflows or its reciprocal is below the normal range (g < -87).
__device__ __forceinline__ float silu(float g) { return g * reciprocal(1.0f + exp_fast(-g)); }

// erf-GELU, g Phi(g) with Phi(g) = erfc(-g / sqrt 2) / 2. For g < 0 Phi is small
// and is computed as such: 1 + erf would leave its rounding error, 2^-24, of
// it (at -5, where Phi is 3e-7, a fifth). With t = 1 / (1 + 0.2975 |g|),
//
//   Phi(-|g|) exp(g^2 / 2) = P(t),
//
// P of degree 6 fitted here in the Chebyshev nodes of t for 0 <= |g| <= 13.3
// by weighted least squares, the weights scaled by the errors until these are
// even: 1.43e-6 relative. With the roundings of FP32, the reciprocal and the
// exponent the result is right to 2^-18 + g^2 2^-23 of itself, down to -13.2,
// where exp is below the normal range and the result is 0. As many
// instructions as the sum with erf (8-bit 300x512x4096 8.60 us for 8.64, FP16
// 333x1008x2731 11.12 for 11.02).
__device__ __forceinline__ float gelu(float g) {
  const float t = reciprocal(fmaf(0.2975f, fabsf(g), 1.0f));
  float poly = fmaf(-0.08747842209f, t, 0.2578530828f);
  poly = fmaf(poly, t, -0.06899382892f);
  poly = fmaf(poly, t, 0.1758866973f);
  poly = fmaf(poly, t, 0.1019707022f);
  poly = fmaf(poly, t, 0.1208796454f);
  poly = fmaf(poly, t, -0.0001185836975f);
  // exp(-g^2 / 2) = 2^(-g^2 log2(e) / 2)
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -0.7213475204f * g));
  const float tail = poly * e;  // Phi(-|g|)
  // Phi(g) is tail or 1 - tail; __fsub_rn is not contracted, so that every
  // kernel rounds alike.
  return g * fabsf(__fsub_rn(tail, g < 0.0f ? 0.0f : 1.0f));
}

// Every form takes the activation from here, so that a token's result does not
// depend on how many rows run beside it (but for the order of FP32 sums).
__device__ __forceinline__ float gated(float gate, float up, int activation) {
  return (activation == kSilu ? silu(gate) : gelu(gate)) * up;
}

// acc is the exact sum of 8-bit products; FP32 keeps 24 of its bits, more
// than the FP16 result. The scales are multiplied first: their product is the
// same for every kernel form, so all forms round alike. They are read by plain
// loads, not through the read-only path, whose memory has to be constant while
// the grid runs: the kernel that writes them may still be running when it starts.
__device__ __forceinline__ float dequantized(int acc, float row_scale, float column_scale, float bias) {
  return fmaf(static_cast<float>(acc), row_scale * column_scale, bias);
}

}  // namespace ctb
