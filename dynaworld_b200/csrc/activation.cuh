// Activations of the matrix product's epilogue and their derivatives, in float.
#pragma once

#include "gsb200.h"

namespace gsb {

constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kSqrt2OverPi = 0.79788456080286536f;
constexpr float kGeluCubic = 0.044715f;

// ReLU passes a NaN on, as torch does.
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == GSB_ACT_RELU) {
    return z < 0.0f ? 0.0f : z;
  } else if constexpr (ACT == GSB_ACT_GELU) {
    return 0.5f * z * (1.0f + erff(z * kSqrtHalf));
  } else if constexpr (ACT == GSB_ACT_GELU_TANH) {
    return 0.5f * z * (1.0f + tanhf(kSqrt2OverPi * fmaf(kGeluCubic * z * z, z, z)));
  } else if constexpr (ACT == GSB_ACT_SILU) {
    return z / (1.0f + expf(-z));
  } else {
    return z;
  }
}

template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == GSB_ACT_RELU) {
    return z <= 0.0f ? 0.0f : 1.0f;
  } else if constexpr (ACT == GSB_ACT_GELU) {
    return fmaf(z * kInvSqrt2Pi, expf(-0.5f * z * z), 0.5f * (1.0f + erff(z * kSqrtHalf)));
  } else if constexpr (ACT == GSB_ACT_GELU_TANH) {
    const float t = tanhf(kSqrt2OverPi * fmaf(kGeluCubic * z * z, z, z));
    return 0.5f * (1.0f + t) + 0.5f * z * (1.0f - t * t) * kSqrt2OverPi * fmaf(3.0f * kGeluCubic * z, z, 1.0f);
  } else if constexpr (ACT == GSB_ACT_SILU) {
    const float s = 1.0f / (1.0f + expf(-z));
    return s * fmaf(z, 1.0f - s, 1.0f);
  } else {
    return 1.0f;
  }
}

}  // namespace gsb
