// Activations of the dense layer and their derivatives, on float32 sums (dense.cu,
// few_rows.cu, linear.cu).
#pragma once

#include "layers_common.cuh"

namespace so3lr_b200 {

constexpr float kInvSqrt2 = 0.70710678f, kInvSqrt2Pi = 0.39894228f;
constexpr float kTanhSlope = 1.5957691f, kTanhCube = 0.044715f;  // 2 sqrt(2 / pi)

// gelu: z Phi(z), Phi through CUDA's erff, within 2^-22 |z|. gelu_tanh: z (1 + tanh(u)) / 2 =
// z sigmoid(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3). relu keeps a NaN.
template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if (ACT == SO3LR_SILU) return silu_f32(z);
  if (ACT == SO3LR_GELU) return z * fmaf(0.5f, erff(z * kInvSqrt2), 0.5f);
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
  if (ACT == SO3LR_GELU)
    return fmaf(z * kInvSqrt2Pi, __expf(-0.5f * z * z), fmaf(0.5f, erff(z * kInvSqrt2), 0.5f));
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
