// Activations of the dense layer and their derivatives, on float32 sums (dense.cu,
// few_rows.cu, linear.cu).
#pragma once

#include "layers_common.cuh"

namespace so3lr_b200 {

constexpr float kInvSqrt2Pi = 0.39894228f;
constexpr float kTanhSlope = 1.5957691f, kTanhCube = 0.044715f;  // 2 sqrt(2 / pi)

// Phi(z), the normal distribution's, and e = exp(-z^2 / 2): Phi(-|z|) = t poly(t) e / 2, t = 1 / (1 +
// p |z| / sqrt 2) (Abramowitz and Stegun 7.1.26, off by 1.5e-7 at most; with erff 24000 x 256 ->
// 1024 takes 49 us, so 38).
__device__ __forceinline__ float normal_cdf(float z, float &e) {
  const float a = fabsf(z);
  float t;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.3275911f * 0.70710678f, a, 1.0f)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * z * (-0.5f * 1.4426950408889634f)));
  float q = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
  q = fmaf(q, t, 0.5f * 1.421413741f);
  q = fmaf(q, t, 0.5f * -0.284496736f);
  q = fmaf(q, t, 0.5f * 0.254829592f) * t * e;
  return z < 0.0f ? q : 1.0f - q;
}
// gelu: z Phi(z). gelu_tanh: z (1 + tanh(u)) / 2 = z sigmoid(2 u), u = sqrt(2 / pi) (z + 0.044715
// z^3). relu keeps a NaN.
template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if (ACT == SO3LR_SILU) return silu_f32(z);
  if (ACT == SO3LR_GELU) {
    float e;
    return z * normal_cdf(z, e);
  }
  if (ACT == SO3LR_GELU_TANH) return z * sigmoid_f32(kTanhSlope * fmaf(kTanhCube * z * z, z, z));
  if (ACT == SO3LR_RELU) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(z) : "f"(0.0f));
    return z;
  }
  return z;
}
// The derivative at a finite z or a NaN.
template <int ACT>
__device__ __forceinline__ float slope(float z) {
  if (ACT == SO3LR_SILU) {
    const float s = sigmoid_f32(z);
    return s * fmaf(z, 1.0f - s, 1.0f);
  }
  if (ACT == SO3LR_GELU) {
    float e;
    const float cdf = normal_cdf(z, e);
    return fmaf(z * kInvSqrt2Pi, e, cdf);
  }
  if (ACT == SO3LR_GELU_TANH) {
    const float s = sigmoid_f32(kTanhSlope * fmaf(kTanhCube * z * z, z, z));
    // beyond 1000 s (1 - s) is 0, and the square would become infinite
    const float c = fminf(fmaxf(z, -1000.0f), 1000.0f);
    return fmaf(c * kTanhSlope * fmaf(3.0f * kTanhCube * c, c, 1.0f), s * (1.0f - s), s);
  }
  if (ACT == SO3LR_RELU) return z > 0.0f ? 1.0f : z <= 0.0f ? 0.0f : z;
  return 1.0f;
}
// z as it is kept for the backward pass, rounded to the element type: its derivative is then off
// by at most half a unit of z, as much as the rounding of dz itself. Kept finite, where every
// derivative has its limit; a NaN stays one.
template <class T>
__device__ __forceinline__ uint32_t kept(float a, float b) {
  uint32_t r;
  if (std::is_same<T, __half>::value)
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <class T>
__device__ __forceinline__ T kept(float z) {
  const uint32_t r = kept<T>(z, 0.0f);
  return *reinterpret_cast<const T *>(&r);
}
// f(std::integral_constant activation)
template <class F>
__device__ __forceinline__ void by_activation(int act, F &&f) {
  switch (act) {
    case SO3LR_SILU: return f(std::integral_constant<int, SO3LR_SILU>{});
    case SO3LR_GELU: return f(std::integral_constant<int, SO3LR_GELU>{});
    case SO3LR_GELU_TANH: return f(std::integral_constant<int, SO3LR_GELU_TANH>{});
    case SO3LR_RELU: return f(std::integral_constant<int, SO3LR_RELU>{});
    default: return f(std::integral_constant<int, SO3LR_NO_ACTIVATION>{});
  }
}

}  // namespace so3lr_b200
