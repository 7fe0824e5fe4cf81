// Activations of the matrix product's epilogue and their derivatives, in float.
//
// They are evaluated for every value of a tile between two tiles' products, so instructions count:
// one exponential and one reciprocal each.  The normal distribution function follows Abramowitz
// and Stegun, Handbook of Mathematical Functions, 7.1.26 (erf within 1.5e-7), whose exponential
// is the density's own; the tanh form of GELU is z sigmoid(2 u).  With the erff / expf / divide
// forms the bf16 product of 16384 x 1024 x 4096 with GELU took 218 us and dz 136 us.
#pragma once

#include "gsb200.h"

namespace gsb {

constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kSqrt2OverPi = 0.79788456080286536f;
constexpr float kGeluCubic = 0.044715f;
constexpr float kLog2E = 1.4426950408889634f;

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Phi(-|z|) and exp(-z^2 / 2): 7.1.26 with its coefficients halved and its argument |z| / sqrt(2).
__device__ __forceinline__ float normal_tail(float z, float& gauss) {
  const float t = fast_rcp(fmaf(0.3275911f * 0.70710678118654752f, fabsf(z), 1.0f));
  float p = fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
  p = fmaf(p, t, 0.5f * 1.421413741f);
  p = fmaf(p, t, 0.5f * -0.284496736f);
  p = fmaf(p, t, 0.5f * 0.254829592f);
  gauss = fast_exp2(z * z * (-0.5f * kLog2E));
  return p * t * gauss;
}

__device__ __forceinline__ float sigmoid_of(float z) { return fast_rcp(1.0f + fast_exp2(-kLog2E * z)); }

// 2 sqrt(2 / pi) (z + 0.044715 z^3)
__device__ __forceinline__ float gelu_tanh_arg(float z) {
  return z * fmaf(2.0f * kSqrt2OverPi * kGeluCubic * z, z, 2.0f * kSqrt2OverPi);
}

// ReLU passes a NaN on, as torch does.
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == GSB_ACT_RELU) {
    return z < 0.0f ? 0.0f : z;
  } else if constexpr (ACT == GSB_ACT_GELU) {
    float gauss;
    const float tail = normal_tail(z, gauss);
    return fmaf(-fabsf(z), tail, fmaxf(z, 0.0f));  // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
  } else if constexpr (ACT == GSB_ACT_GELU_TANH) {
    return z * sigmoid_of(gelu_tanh_arg(z));
  } else if constexpr (ACT == GSB_ACT_SILU) {
    return z * sigmoid_of(z);
  } else {
    return z;
  }
}

template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == GSB_ACT_RELU) {
    return z <= 0.0f ? 0.0f : 1.0f;
  } else if constexpr (ACT == GSB_ACT_GELU) {
    float gauss;
    const float tail = normal_tail(z, gauss);
    return fmaf(z * kInvSqrt2Pi, gauss, z < 0.0f ? tail : 1.0f - tail);
  } else if constexpr (ACT == GSB_ACT_GELU_TANH) {
    const float s = sigmoid_of(gelu_tanh_arg(z));
    // s (1 - s) is 0 from |z| = 10 on, where z^2 must not overflow
    const float du = fmaf(6.0f * kSqrt2OverPi * kGeluCubic, fminf(z * z, 1e4f), 2.0f * kSqrt2OverPi);
    return fmaf(z * s * (1.0f - s), du, s);
  } else if constexpr (ACT == GSB_ACT_SILU) {
    const float s = sigmoid_of(z);
    return s * fmaf(z, 1.0f - s, 1.0f);
  } else {
    return 1.0f;
  }
}

}  // namespace gsb
