// Activations of gated blocks, in FP32: act(x) and its derivative.
//
//   SiLU       x s,  s = 1 / (1 + e^-x)                    s + x s (1 - s)
//   GELU       x P,  P = erfc(-x / sqrt 2) / 2             P + x e^(-x^2 / 2) / sqrt(2 pi)
//   GELU_TANH  x s(y),  y = 2 sqrt(2 / pi) (x + 0.044715 x^3)   s + x s (1 - s) y'     (the half of 1 + tanh(y / 2) is s(y))
//   RELU       x where x > 0                               1 where x > 0
// P of a negative x is e^(-x^2 / 2) times a function that falls slowly, t times a polynomial in t = 1 / (1 + 0.36 |x| / sqrt 2),
// fitted to 3.5e-8 of erfc's values over all |x|; P(x) = 1 - P(-x).  So it keeps its significant bits for negative x, and its
// derivative has the same exponential.  At minus infinity SiLU and both GELUs are 0 times infinity, NaN, as their formulas say.
#pragma once
#include <cumpsgemm/cumpsgemm_ext.h>
#include <hip/hip_runtime.h>
#include <type_traits>

namespace cumpsgemm_amd {

// EXACT: for FP32 results.  Otherwise the exponential and the reciprocal are the hardware's own, off by a few 2^-23 |x|, which
// a rounding to 16 bits does not show.
template <bool EXACT> __device__ inline float sigmoid(float x) {
  if constexpr (EXACT) return 1.0f / (1.0f + expf(-x));
  else return __builtin_amdgcn_rcpf(1.0f + __expf(-x));
}

// P, and e^(-x^2 / 2)
template <bool EXACT> __device__ inline float normal_below(float x, float &bell) {
  constexpr float c[10] = {0.101554129f, 0.101553861f, 0.0949720355f, 0.081958194f, 0.0614630061f,
                             0.0532569567f, -0.0143161425f, 0.0717105734f, -0.0709835375f, 0.0188309427f};
  const float u = 1.0f + 0.25455844f * fabsf(x), t = EXACT ? 1.0f / u : __builtin_amdgcn_rcpf(u);
  bell = EXACT ? expf(-0.5f * x * x) : __expf(-0.5f * x * x);
  float p = c[9];
#pragma unroll
  for (int i = 8; i >= 0; i--) p = fmaf(p, t, c[i]);
  const float tail = bell * (t * p);
  return x > 0.0f ? 1.0f - tail : tail;
}

// act(x), and its derivative as slope if DERIVATIVE
template <uint32_t ACT, bool EXACT, bool DERIVATIVE> __device__ inline float activation(float x, float &slope) {
  if constexpr (ACT == CUMPSGEMM_SILU) {
    const float s = sigmoid<EXACT>(x), y = x * s;
    if (DERIVATIVE) slope = fmaf(y, 1.0f - s, s);
    return y;
  } else if constexpr (ACT == CUMPSGEMM_GELU) {
    float bell;
    const float p = normal_below<EXACT>(x, bell);
    if (DERIVATIVE) slope = fmaf(x * 0.39894228f, bell, p);
    return x * p;
  } else if constexpr (ACT == CUMPSGEMM_GELU_TANH) {
    const float s = sigmoid<EXACT>(1.5957691216f * (x + 0.044715f * x * x * x)), y = x * s;
    if (DERIVATIVE) slope = fmaf(y * (1.0f - s), 1.5957691216f * (1.0f + 0.134145f * x * x), s);
    return y;
  } else {
    if (DERIVATIVE) slope = x > 0.0f ? 1.0f : 0.0f;
    return x < 0.0f ? 0.0f : x; // (a NaN stays one)
  }
}
// f(the activation, as a constant)
template <class F> __device__ inline void with_activation(uint32_t act, F f) {
  if (act == CUMPSGEMM_SILU) f(std::integral_constant<uint32_t, CUMPSGEMM_SILU>{});
  else if (act == CUMPSGEMM_GELU) f(std::integral_constant<uint32_t, CUMPSGEMM_GELU>{});
  else if (act == CUMPSGEMM_GELU_TANH) f(std::integral_constant<uint32_t, CUMPSGEMM_GELU_TANH>{});
  else f(std::integral_constant<uint32_t, CUMPSGEMM_RELU>{});
}

} // namespace cumpsgemm_amd
