// Activations of the linear layer's epilogue, in fp32. SiLU's sigmoid is the one of
// swiglu_math.h; the other two are written so that their tails keep their relative
// accuracy: gelu by the normal distribution's lower tail (0.5 (1 + erf) cancels for
// negative z), gelu_tanh by 0.5 (1 + tanh v) = sigmoid(2 v).
//
// The lower tail is Phi(-a) = 0.5 exp(-a^2 / 2) erfcx(a / sqrt 2), a >= 0, with the
// scaled complementary error function as t p(t), t = 1 / (1 + 0.375 a / sqrt 2), p of
// degree 8 fitted to it by reweighted least squares in t (largest relative error with the
// coefficients below 1.6e-8 up to a = 14.8, past which the product underflows, 4e-8 with
// their fp32 values; the function's own, in fp32, is 5e-7 up to a = 1, 2e-6 up to 6 and
// 8e-6 up to 12.9, as the rounding of the exponent counts a^2 times; the hardware's
// reciprocal and exponential add a step each). One exponential, which the
// derivative's density shares, one reciprocal and ten multiplications; with the math
// library's erfc, whose branches a wave takes both of, the product of [8192, 1152] x 4304
// with this epilogue takes 150 us instead of 123 (110 without an activation).
#pragma once

#include "swiglu_math.h"

namespace mla {

enum : int { kActNone = 0, kActSilu = 1, kActGelu = 2, kActGeluTanh = 3 };

constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kGeluC = 1.5957691216057308f;   // 2 sqrt(2 / pi)
constexpr float kGeluC3 = 0.07135481627262735f; // 0.044715 times that

// Beyond 30 the derivatives are 0 or 1 to the last bit, and z^2, z^3 stay finite.
constexpr float kActFar = 30.f;

// Phi(z), and e = exp(-z^2 / 2).
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float t = __builtin_amdgcn_rcpf(1.0f + 0.26516504294495532f * fabsf(z));
  e = __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z);
  float p = 0.5f * 0.0609968481f;
  p = p * t - 0.5f * 0.284775211f;
  p = p * t + 0.5f * 0.427277103f;
  p = p * t - 0.5f * 0.223726358f;
  p = p * t + 0.5f * 0.269907342f;
  p = p * t + 0.5f * 0.123087606f;
  p = p * t + 0.5f * 0.204918483f;
  p = p * t + 0.5f * 0.210703824f;
  p = p * t + 0.5f * 0.211610354f;
  const float tail = e * (p * t);
  return z < 0.f ? tail : 1.0f - tail;
}

template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (ACT == kActSilu) {
    return z * sigmoid_f(z);
  } else if constexpr (ACT == kActGelu) {
    float e;
    return z * normal_cdf(z, e);
  } else if constexpr (ACT == kActGeluTanh) {
    return z * sigmoid_f(z * (kGeluC + kGeluC3 * z * z));
  } else {
    return z;
  }
}

template <int ACT>
__device__ __forceinline__ float act_grad(float z) {
  if constexpr (ACT == kActSilu) {
    const float s = sigmoid_f(z);
    return s * (1.0f + z * (1.0f - s));
  } else if constexpr (ACT == kActGelu) {
    if (fabsf(z) > kActFar) return z > 0.f ? 1.f : 0.f;
    float e;
    const float c = normal_cdf(z, e);
    return c + z * kInvSqrt2Pi * e;
  } else if constexpr (ACT == kActGeluTanh) {
    if (fabsf(z) > kActFar) return z > 0.f ? 1.f : 0.f;
    const float s = sigmoid_f(z * (kGeluC + kGeluC3 * z * z));
    return s + z * s * (1.0f - s) * (kGeluC + 3.0f * kGeluC3 * z * z);
  } else {
    return 1.f;
  }
}

}  // namespace mla
