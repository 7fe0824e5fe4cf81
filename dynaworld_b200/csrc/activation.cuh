// Activations of the matrix product's epilogue and their derivatives, in float.
//
// They are evaluated for every value of a tile between two tiles' products, so instructions count:
// one exponential and one reciprocal each.  The normal distribution function is the density's own
// exponential times a polynomial in t = 1 / (1 + c |z|): for 16-bit outputs Abramowitz and Stegun, Handbook
// of Mathematical Functions, 7.1.26 (erf within 1.5e-7, which in the tail is 5e-5 of the value at z = -3),
// for float outputs (FINE) three degrees more of the same form (4,096 x 512 x 2,560 float with GELU: 64 us
// with 7.1.26, 66 so).  The tanh form of GELU is z sigmoid(2 u).
// With the erff / expf / divide forms the bf16 product of 16384 x 1024 x 4096 with GELU took 218 us and dz
// 136 us.
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

// Two floats in one register pair: the FMA pipe takes both in one instruction (sm_100).
struct F2 {
  unsigned long long v;
  F2() = default;
  __device__ __forceinline__ explicit F2(float both) : F2(both, both) {}
  __device__ __forceinline__ F2(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ void get(float& lo, float& hi) const {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
  }
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
template <typename F>
__device__ __forceinline__ F2 each(F2 a, F f) {
  float lo, hi;
  a.get(lo, hi);
  return F2(f(lo), f(hi));
}
__device__ __forceinline__ F2 exp2_2(F2 a) { return each(a, [](float x) { return fast_exp2(x); }); }
__device__ __forceinline__ F2 rcp_2(F2 a) { return each(a, [](float x) { return fast_rcp(x); }); }

// -|z|, Phi(-|z|) and exp(-z^2 / 2).  7.1.26 with its coefficients halved, its argument |z| / sqrt(2).
// FINE: minimax fit of Phi(-a) / (t exp(-a^2 / 2)) over a <= 13.5 (where the exponential leaves float's
// range) by its relative error, 9.4e-8, with the c that a search found best for the degree.
template <bool FINE>
__device__ __forceinline__ F2 normal_tail(F2 z, F2& minus, F2& gauss) {
  minus = each(z, [](float x) { return __int_as_float(__float_as_int(x) | 0x80000000); });
  const F2 t = rcp_2(fma2(F2(FINE ? -0.305f : -0.3275911f * 0.70710678118654752f), minus, F2(1.0f)));
  F2 p;
  if constexpr (FINE) {
    p = fma2(F2(0.0366991855f), t, F2(-0.1529882908f));
    p = fma2(p, t, F2(0.1857168636f));
    p = fma2(p, t, F2(-0.0379767906f));
    p = fma2(p, t, F2(0.1210216580f));
    p = fma2(p, t, F2(0.1034208725f));
    p = fma2(p, t, F2(0.1224668160f));
    p = fma2(p, t, F2(0.1216397327f));
  } else {
    p = fma2(F2(0.5f * 1.061405429f), t, F2(0.5f * -1.453152027f));
    p = fma2(p, t, F2(0.5f * 1.421413741f));
    p = fma2(p, t, F2(0.5f * -0.284496736f));
    p = fma2(p, t, F2(0.5f * 0.254829592f));
  }
  gauss = exp2_2(mul2(mul2(z, z), F2(-0.5f * kLog2E)));
  return mul2(mul2(p, t), gauss);
}

__device__ __forceinline__ F2 sigmoid_of(F2 z) { return rcp_2(add2(exp2_2(mul2(z, F2(-kLog2E))), F2(1.0f))); }

// 2 sqrt(2 / pi) (z + 0.044715 z^3), from z and z^2
__device__ __forceinline__ F2 gelu_tanh_arg(F2 z, F2 zz) {
  return mul2(z, fma2(F2(2.0f * kSqrt2OverPi * kGeluCubic), zz, F2(2.0f * kSqrt2OverPi)));
}

// ReLU passes a NaN on, as torch does.
template <int ACT, bool FINE>
__device__ __forceinline__ F2 act_value(F2 z) {
  if constexpr (ACT == GSB_ACT_RELU) {
    return each(z, [](float x) { return x < 0.0f ? 0.0f : x; });
  } else if constexpr (ACT == GSB_ACT_GELU) {
    // z Phi(z) = max(z, 0) - |z| Phi(-|z|), whose second term is 0 from z = 15 on: there |z| ends at 1e4, so
    // that +infinity does not meet that 0 (-infinity does: NaN, as z Phi(z) is)
    F2 minus, gauss;
    const F2 tail = normal_tail<FINE>(each(z, [](float x) { return fminf(x, 1e4f); }), minus, gauss);
    return fma2(minus, tail, each(z, [](float x) { return fmaxf(x, 0.0f); }));
  } else if constexpr (ACT == GSB_ACT_GELU_TANH) {
    return mul2(z, sigmoid_of(gelu_tanh_arg(z, mul2(z, z))));
  } else if constexpr (ACT == GSB_ACT_SILU) {
    return mul2(z, sigmoid_of(z));
  } else {
    return z;
  }
}

template <int ACT, bool FINE>
__device__ __forceinline__ F2 act_slope(F2 z) {
  if constexpr (ACT == GSB_ACT_RELU) {
    return each(z, [](float x) { return x <= 0.0f ? 0.0f : 1.0f; });
  } else if constexpr (ACT == GSB_ACT_GELU) {
    F2 minus, gauss;
    const F2 tail = normal_tail<FINE>(z, minus, gauss);
    float z0, z1, h0, h1;
    z.get(z0, z1);
    F2 cdf;
    if constexpr (FINE) {
      float t0, t1;
      tail.get(t0, t1);
      fma2(tail, F2(-1.0f), F2(1.0f)).get(h0, h1);
      cdf = F2(z0 < 0.0f ? t0 : h0, z1 < 0.0f ? t1 : h1);
    } else {  // Phi(z) = 1/2 + (1/2 - Phi(-|z|)) with the sign of z
      fma2(tail, F2(-1.0f), F2(0.5f)).get(h0, h1);
      cdf = add2(F2(copysignf(h0, z0), copysignf(h1, z1)), F2(0.5f));
    }
    return fma2(mul2(z, F2(kInvSqrt2Pi)), gauss, cdf);
  } else if constexpr (ACT == GSB_ACT_GELU_TANH) {
    const F2 zz = mul2(z, z);
    const F2 s = sigmoid_of(gelu_tanh_arg(z, zz));
    // s (1 - s) is 0 from |z| = 10 on, where z^2 must not overflow
    const F2 du = fma2(F2(6.0f * kSqrt2OverPi * kGeluCubic), each(zz, [](float x) { return fminf(x, 1e4f); }),
                       F2(2.0f * kSqrt2OverPi));
    return fma2(mul2(z, mul2(s, fma2(s, F2(-1.0f), F2(1.0f)))), du, s);
  } else if constexpr (ACT == GSB_ACT_SILU) {
    const F2 s = sigmoid_of(z);
    return mul2(s, fma2(z, fma2(s, F2(-1.0f), F2(1.0f)), F2(1.0f)));
  } else {
    return F2(1.0f);
  }
}

// V values at once, for outputs of type O.
template <int ACT, typename O, int V>
__device__ __forceinline__ void apply_value(float (&z)[V]) {
  constexpr bool FINE = sizeof(O) == 4;
  if constexpr (ACT != GSB_ACT_NONE) {
#pragma unroll
    for (int u = 0; u < V; u += 2) {
      float unused;
      if (u + 1 < V) act_value<ACT, FINE>(F2(z[u], z[u + 1])).get(z[u], z[u + 1]);
      else act_value<ACT, FINE>(F2(z[u], 0.0f)).get(z[u], unused);
    }
  }
}
template <int ACT, typename O, int V>
__device__ __forceinline__ void apply_slope(float (&z)[V]) {
  constexpr bool FINE = sizeof(O) == 4;
#pragma unroll
  for (int u = 0; u < V; u += 2) {
    float unused;
    if (u + 1 < V) act_slope<ACT, FINE>(F2(z[u], z[u + 1])).get(z[u], z[u + 1]);
    else act_slope<ACT, FINE>(F2(z[u], 0.0f)).get(z[u], unused);
  }
}

}  // namespace gsb
