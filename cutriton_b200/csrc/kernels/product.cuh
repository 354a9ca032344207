// Epilogue arithmetic of the gated and 8-bit products, in FP32; each output is
// rounded to FP16 once, by the caller.
#pragma once

#include "common.cuh"

namespace ctb {

enum : int { kSilu = 0, kGelu = 1 };

// g / (1 + exp(-g)); the denominator overflows to infinity below -88, where
// the result is -0 to FP32's precision.
__device__ __forceinline__ float silu(float g) { return g / (1.0f + __expf(-g)); }

// silu with an approximate division (2 ulp; 0 where the denominator passes
// 2^126, as the quotient rounds to there in FP16).
__device__ __forceinline__ float silu_fast(float g) { return __fdividef(g, 1.0f + __expf(-g)); }

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
