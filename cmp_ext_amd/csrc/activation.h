// Activations of gated blocks and their derivatives, in fp32.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/cmpext3_projection.h"

namespace cmpext3 {

// 1 / (1 + exp(-x)) on the hardware's 2^x and reciprocal: off by 2^-22 of itself for |x| < 8, by
// |x| 2^-24 more beyond, where the argument's rounding counts; both are far below the 16 bits
// that results are held in.  The functions with every last bit cost a prompt's product 3 %.
__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * x));
}
// P(Z <= g): by erfc, since 1 + erf loses the digits of negative g.
__device__ __forceinline__ float normal_cdf(float g) { return 0.5f * erfcf(-0.70710678f * g); }
constexpr float kGeluTanh = 1.59576912f;  // 2 sqrt(2 / pi): 1 + tanh(y) = 2 sigmoid(2 y)

template <int ACT>
__device__ __forceinline__ float act_value(float g) {
  if constexpr (ACT == CMPEXT3_ACT_SILU) return g * sigmoid(g);
  if constexpr (ACT == CMPEXT3_ACT_GELU) return g * normal_cdf(g);
  if constexpr (ACT == CMPEXT3_ACT_GELU_TANH) return g * sigmoid(kGeluTanh * (g + 0.044715f * g * g * g));
  return g <= 0.f ? 0.f : g;  // relu; NaN stays
}

// The value and the derivative.  Past |g| = 64 every derivative is 0 or 1 to the last bit; the
// bound keeps powers of g from overflowing against a factor of zero.
template <int ACT>
__device__ __forceinline__ void act_both(float g, float& value, float& slope) {
  const float b = fminf(fmaxf(g, -64.f), 64.f);
  if constexpr (ACT == CMPEXT3_ACT_SILU) {
    const float s = sigmoid(g);
    value = g * s;
    slope = s * (1.f + b * (1.f - s));
  } else if constexpr (ACT == CMPEXT3_ACT_GELU) {
    const float s = normal_cdf(g);
    value = g * s;
    slope = s + b * (0.39894228f * __builtin_amdgcn_exp2f(-0.72134752f * b * b));
  } else if constexpr (ACT == CMPEXT3_ACT_GELU_TANH) {
    const float s = sigmoid(kGeluTanh * (g + 0.044715f * g * g * g));
    value = g * s;
    slope = s + b * s * (1.f - s) * (kGeluTanh * (1.f + 0.134145f * b * b));
  } else {
    value = g <= 0.f ? 0.f : g;
    slope = g <= 0.f ? 0.f : g != g ? g : 1.f;
  }
  if (g != g) slope = g;  // the bound's maximum drops a NaN
}

// f(std::integral_constant<int, ACT>) for the activation of a call (uniform over its workgroups).
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case CMPEXT3_ACT_SILU: return f(std::integral_constant<int, CMPEXT3_ACT_SILU>{});
    case CMPEXT3_ACT_GELU: return f(std::integral_constant<int, CMPEXT3_ACT_GELU>{});
    case CMPEXT3_ACT_GELU_TANH: return f(std::integral_constant<int, CMPEXT3_ACT_GELU_TANH>{});
    default: return f(std::integral_constant<int, CMPEXT3_ACT_RELU>{});
  }
}

}  // namespace cmpext3
