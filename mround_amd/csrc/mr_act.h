// The activations of an ungated MLP and their derivatives, in fp32.
#pragma once

#include "mr_common.h"

namespace mr {

// The upper tail of the normal distribution at a >= 0, from e = exp(-a^2 / 2):
// e times a polynomial in t = 1 / (1 + 0.3 a), the form of Abramowitz and Stegun's
// 7.1.26, with eight coefficients fitted here to erfcx(a / sqrt 2) / 2 over 0 .. 14
// (1.5e-7 of the value, 4.5e-7 in fp32). From it x Phi(x) keeps its digits for
// negative x, where 1 + erf has none left, for 17 instructions of which two are
// transcendental.
__device__ __forceinline__ float normal_tail(float a, float e) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3f, a, 1.0f));
  float r = 0.03567483648657799f;
  r = __builtin_fmaf(r, t, -0.1572033166885376f);
  r = __builtin_fmaf(r, t, 0.20635385811328888f);
  r = __builtin_fmaf(r, t, -0.05368392914533615f);
  r = __builtin_fmaf(r, t, 0.12856176495552063f);
  r = __builtin_fmaf(r, t, 0.09991345554590225f);
  r = __builtin_fmaf(r, t, 0.12075395882129669f);
  r = __builtin_fmaf(r, t, 0.11962930113077164f);
  return r * t * e;
}

// exp(-a^2 / 2)
__device__ __forceinline__ float half_square_exp(float a) {
  return __builtin_amdgcn_exp2f(a * a * -0.72134752044448170368f);
}

// x Phi(x) by the tanh approximation is x sigmoid(2 u), u = sqrt(2 / pi) (x + 0.044715 x^3).
__device__ __forceinline__ float tanh_gelu_arg(float x) {
  return x * __builtin_fmaf(x * x, 0.071354816272600247f, 1.5957691216057308f);  // 2 u
}

template <int F>
__device__ __forceinline__ float activate(float x) {
  if constexpr (F == MR_ACT_RELU) {
    return x < 0.0f ? 0.0f : x;  // (NaN passes)
  } else if constexpr (F == MR_ACT_RELU2) {
    const float r = x < 0.0f ? 0.0f : x;
    return r * r;
  } else if constexpr (F == MR_ACT_SILU) {
    return silu(x);
  } else if constexpr (F == MR_ACT_GELU) {
    const float a = __builtin_fabsf(x), q = normal_tail(a, half_square_exp(a));
    return x * (x < 0.0f ? q : 1.0f - q);
  } else {
    return x * sigmoid(tanh_gelu_arg(x));
  }
}

// The derivative, with relu's zero at zero.
template <int F>
__device__ __forceinline__ float activate_slope(float x) {
  if constexpr (F == MR_ACT_RELU) {
    return x <= 0.0f ? 0.0f : 1.0f;
  } else if constexpr (F == MR_ACT_RELU2) {
    return x <= 0.0f ? 0.0f : 2.0f * x;
  } else if constexpr (F == MR_ACT_SILU) {
    const float s = sigmoid(x);
    return s * __builtin_fmaf(x, 1.0f - s, 1.0f);
  } else if constexpr (F == MR_ACT_GELU) {
    const float a = __builtin_fabsf(x), e = half_square_exp(a), q = normal_tail(a, e);
    return __builtin_fmaf(x, e * 0.39894228040143267794f, x < 0.0f ? q : 1.0f - q);
  } else {
    // s + x s (1 - s) (2 u)'; past 12 the second term is below 1e-38, and its factors' product no number
    const float c = clampf(x, -12.0f, 12.0f), s = sigmoid(tanh_gelu_arg(x));
    const float du = __builtin_fmaf(c * c, 3.0f * 0.071354816272600247f, 1.5957691216057308f);
    return __builtin_fmaf(c * s, (1.0f - s) * du, s);
  }
}

}  // namespace mr
