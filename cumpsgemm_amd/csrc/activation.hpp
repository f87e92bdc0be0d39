// Activations of gated blocks, in FP32: act(x) and its derivative.
//
//   SiLU       x s,  s = 1 / (1 + e^-x)                    s + x s (1 - s)
//   GELU       x P,  P = erfc(-x / sqrt 2) / 2             P + x e^(-x^2 / 2) / sqrt(2 pi)
//   GELU_TANH  x s(y),  y = 2 sqrt(2 / pi) (x + 0.044715 x^3)   s + x s (1 - s) y'     (the half of 1 + tanh(y / 2) is s(y))
//   RELU       x where x > 0                               1 where x > 0
// P of a negative x is e^(-x^2 / 2) times a function that falls slowly, t times a polynomial in t = 1 / (1 + 0.36 |x| / sqrt 2),
// fitted to 3.5e-8 of erfc's values over all |x|; P(x) = 1 - P(-x).  So it keeps its significant bits for negative x, and its
// derivative has the same exponential.  At the infinities, where the formulas have 0 times infinity, all of them have their limits: a
// projection that FP16 could only store as an infinity has a gradient like any other far out.  (NaN stays NaN.)
#pragma once
#include <cumpsgemm/cumpsgemm_ext.h>
#include <hip/hip_runtime.h>
#include <type_traits>

namespace cumpsgemm_amd {

// EXACT: for FP32 results, off by a few 2^-24.  Otherwise the exponential and the reciprocal are the hardware's own, off by a
// few 2^-23 |x|, which a rounding to 16 bits does not show.
// e^x for x up to 88 (from there on: e^88), 0 below -150
template <bool EXACT> __device__ inline float exponential(float x) {
  if constexpr (!EXACT) return __expf(x);
  constexpr float log2e = 1.44269504f, rest = 1.92596299e-8f, ln2 = 0.693147181f;
  x = fminf(fmaxf(x, -150.0f), 88.0f);
  // (x log2 e in two parts, the second of which the hardware's 2^t does not see)
  const float t = x * log2e, more = fmaf(x, rest, fmaf(x, log2e, -t));
  const float y = __builtin_amdgcn_exp2f(t);
  return fmaf(y, more * ln2, y);
}
// 1 / x, x from 1 to e^88 + 1
template <bool EXACT> __device__ inline float reciprocal(float x) {
  const float r = __builtin_amdgcn_rcpf(x);
  return EXACT ? fmaf(fmaf(-x, r, 1.0f), r, r) : r;
}
template <bool EXACT> __device__ inline float sigmoid(float x) {
  const float s = reciprocal<EXACT>(1.0f + exponential<EXACT>(-x));
  return EXACT && x < -88.0f ? 0.0f : s; // (6e-39 from there on otherwise, times an x of -1e38)
}

// P, and e^(-x^2 / 2)
template <bool EXACT> __device__ inline float normal_below(float x, float &bell) {
  constexpr float c[10] = {0.101554129f, 0.101553861f, 0.0949720355f, 0.081958194f, 0.0614630061f,
                           0.0532569567f, -0.0143161425f, 0.0717105734f, -0.0709835375f, 0.0188309427f};
  const float t = reciprocal<EXACT>(1.0f + 0.25455844f * fminf(fabsf(x), 1e30f));
  bell = exponential<EXACT>(-0.5f * x * x);
  float p = c[9];
#pragma unroll
  for (int i = 8; i >= 0; i--) p = fmaf(p, t, c[i]);
  const float tail = bell * (t * p);
  return x > 0.0f ? 1.0f - tail : tail;
}

// act(x), and its derivative as slope if DERIVATIVE
template <uint32_t ACT, bool EXACT, bool DERIVATIVE> __device__ inline float activation(float x, float &slope) {
  // (values that minus infinity and infinity are taken as, where the other factor is 0; unlike fmaxf and fminf these keep a NaN)
  constexpr float least = -3.4028235e38f, far = 1000.0f;
  if constexpr (ACT != CUMPSGEMM_RELU) x = __builtin_elementwise_maximum(x, least);
  if constexpr (ACT == CUMPSGEMM_SILU) {
    const float s = sigmoid<EXACT>(x), y = x * s;
    if (DERIVATIVE) slope = fmaf(__builtin_elementwise_minimum(y, far), 1.0f - s, s);
    return y;
  } else if constexpr (ACT == CUMPSGEMM_GELU) {
    float bell;
    const float p = normal_below<EXACT>(x, bell);
    if (DERIVATIVE) slope = fmaf(__builtin_elementwise_minimum(x, far) * 0.39894228f, bell, p);
    return x * p;
  } else if constexpr (ACT == CUMPSGEMM_GELU_TANH) {
    const float s = sigmoid<EXACT>(1.5957691216f * (x + 0.044715f * x * x * x)), y = x * s;
    // (y (1 - s) is 0 long before `far`, and stays so where x^2 is infinite)
    const float near = fminf(fmaxf(x, -far), far);
    if (DERIVATIVE) slope = fmaf(__builtin_elementwise_minimum(y, far) * (1.0f - s), 1.5957691216f * (1.0f + 0.134145f * near * near), s);
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
