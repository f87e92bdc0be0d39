// Activations of gated blocks, in FP32: act(x) and its derivative.
//
//   SiLU       x s,  s = 1 / (1 + e^-x)                    s + x s (1 - s)
//   GELU       x P,  P = erfc(-x / sqrt 2) / 2             P + x e^(-x^2 / 2) / sqrt(2 pi)
//   GELU_TANH  x s(y),  y = 2 sqrt(2 / pi) (x + 0.044715 x^3)   s + x s (1 - s) y'     (the half of 1 + tanh(y / 2) is s(y))
//   RELU       x where x > 0                               1 where x > 0
// P comes from erfc, not from 1 + erf, so that it keeps its significant bits for negative x.  At minus infinity SiLU and both
// GELUs are 0 times infinity, NaN, as their formulas say.
#pragma once
#include <cumpsgemm/cumpsgemm_ext.h>
#include <hip/hip_runtime.h>

namespace cumpsgemm_amd {

// EXACT: for FP32 results.  Otherwise the exponential and the reciprocal are the hardware's own, off by a few 2^-23 |x|, which
// a rounding to 16 bits does not show.
template <bool EXACT> __device__ inline float sigmoid(float x) {
  if constexpr (EXACT) return 1.0f / (1.0f + expf(-x));
  else return __builtin_amdgcn_rcpf(1.0f + __expf(-x));
}

// slope: the derivative, if DERIVATIVE
template <bool EXACT, bool DERIVATIVE> __device__ inline float activation(uint32_t act, float x, float &slope) {
  if (act == CUMPSGEMM_SILU) {
    const float s = sigmoid<EXACT>(x);
    if (DERIVATIVE) slope = s + x * s * (1.0f - s);
    return x * s;
  }
  if (act == CUMPSGEMM_GELU) {
    const float p = 0.5f * erfcf(-0.70710678f * x);
    if (DERIVATIVE) slope = p + x * 0.39894228f * (EXACT ? expf(-0.5f * x * x) : __expf(-0.5f * x * x));
    return x * p;
  }
  if (act == CUMPSGEMM_GELU_TANH) {
    const float s = sigmoid<EXACT>(1.5957691216f * (x + 0.044715f * x * x * x));
    if (DERIVATIVE) slope = s + x * s * (1.0f - s) * (1.5957691216f * (1.0f + 0.134145f * x * x));
    return x * s;
  }
  if (DERIVATIVE) slope = x > 0.0f ? 1.0f : 0.0f;
  return x < 0.0f ? 0.0f : x; // (a NaN stays one)
}

} // namespace cumpsgemm_amd
