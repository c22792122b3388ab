// The gates of the gated feed-forward block and their derivatives, in FP32.
//
//   silu        a = g s,  a' = s (1 + g (1 - s)),  s = 1 / (1 + e^-g)
//   gelu        a = g P,  a' = P + g p,  P = erfc(-g / sqrt 2) / 2 (no cancellation for negative g),  p = e^(-g^2/2) / sqrt(2 pi)
//               erfc by the Chebyshev fit of Press et al., Numerical Recipes, section 6.2 (relative error 1.2e-7): half of the instructions of
//               erfcf(), which took 5 us of 22 at 333 x 2056
//   gelu_tanh   a = g s,  a' = s + g s (1 - s) w',  s = sigmoid(w),  w = 2 sqrt(2/pi) (g + 0.044715 g^3): (1 + tanh(w/2)) / 2 = s
//
// __fdividef is off by 2 units in the last place, __expf of an argument t by 2 + 1.17 |t| of them: 2^-21 together near zero, 6e-6 at t = -43 (the
// tail of gelu at g = -9), 1.3e-5 at 88, against up to 2^-8 by the BF16 rounding that follows.  Far from zero the exponential
// overflows to infinity and s becomes an exact 0.
#pragma once
#include <cuda_runtime.h>
#include "../include/fp4ar_layer.h"

namespace fp4ar {

__device__ __forceinline__ float sigmoid_f32(float g) { return __fdividef(1.0f, 1.0f + __expf(-g)); }
__device__ __forceinline__ float gelu_tanh_arg(float g) { return 1.5957691216f * fmaf(0.044715f * g * g, g, g); }

// P(g), the normal distribution
__device__ __forceinline__ float normal_cdf(float g) {
  const float z = fabsf(g) * 0.70710678119f, t = __fdividef(1.0f, fmaf(0.5f, z, 1.0f));
  float e = fmaf(t, 0.17087277f, -0.82215223f);
  e = fmaf(t, e, 1.48851587f);
  e = fmaf(t, e, -1.13520398f);
  e = fmaf(t, e, 0.27886807f);
  e = fmaf(t, e, -0.18628806f);
  e = fmaf(t, e, 0.09678418f);
  e = fmaf(t, e, 0.37409196f);
  e = fmaf(t, e, 1.00002368f);
  e = fmaf(t, e, -1.26551223f);
  const float tail = 0.5f * t * __expf(fmaf(-z, z, e));
  return g < 0.0f ? tail : 1.0f - tail;
}

template <int ACT>
__device__ __forceinline__ float act_value(float g) {
  if constexpr (ACT == FP4AR_ACT_SILU) return g * sigmoid_f32(g);
  else if constexpr (ACT == FP4AR_ACT_GELU) return g * normal_cdf(g);
  else return g * sigmoid_f32(gelu_tanh_arg(g));
}

// value and derivative
template <int ACT>
__device__ __forceinline__ void act_both(float g, float& value, float& slope) {
  if constexpr (ACT == FP4AR_ACT_SILU) {
    const float s = sigmoid_f32(g);
    value = g * s;
    slope = s * fmaf(g, 1.0f - s, 1.0f);
  } else if constexpr (ACT == FP4AR_ACT_GELU) {
    const float P = normal_cdf(g);
    value = g * P;
    slope = fmaf(g, 0.39894228040f * __expf(-0.5f * g * g), P);
  } else {
    const float s = sigmoid_f32(gelu_tanh_arg(g)), t = s * (1.0f - s);
    value = g * s;
    slope = t == 0.0f ? s : fmaf(g * t, 1.5957691216f * fmaf(0.134145f, g * g, 1.0f), s);      // t = 0: g^2 may be infinite
  }
}

}  // namespace fp4ar
