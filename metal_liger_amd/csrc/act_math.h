// Activations of the linear layer's epilogue, in fp32. SiLU's sigmoid is the one of
// swiglu_math.h; the other two are written so that their tails keep their relative
// accuracy: gelu by erfc (0.5 (1 + erf) cancels for negative z), gelu_tanh by
// 0.5 (1 + tanh v) = sigmoid(2 v).
#pragma once

#include "swiglu_math.h"

namespace mla {

enum : int { kActNone = 0, kActSilu = 1, kActGelu = 2, kActGeluTanh = 3 };

constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kGeluC = 1.5957691216057308f;   // 2 sqrt(2 / pi)
constexpr float kGeluC3 = 0.07135481627262735f; // 0.044715 times that

// Beyond 30 the derivatives are 0 or 1 to the last bit, and z^2, z^3 stay finite.
constexpr float kActFar = 30.f;

template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (ACT == kActSilu) {
    return z * sigmoid_f(z);
  } else if constexpr (ACT == kActGelu) {
    return z * (0.5f * erfcf(-z * kSqrtHalf));
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
    return 0.5f * erfcf(-z * kSqrtHalf) +
           z * kInvSqrt2Pi * __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z);
  } else if constexpr (ACT == kActGeluTanh) {
    if (fabsf(z) > kActFar) return z > 0.f ? 1.f : 0.f;
    const float s = sigmoid_f(z * (kGeluC + kGeluC3 * z * z));
    return s + z * s * (1.0f - s) * (kGeluC + 3.0f * kGeluC3 * z * z);
  } else {
    return 1.f;
  }
}

}  // namespace mla
