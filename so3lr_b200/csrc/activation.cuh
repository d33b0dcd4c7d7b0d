// Activations of the dense layer and their derivatives, on float32 sums (dense.cu,
// few_rows.cu, linear.cu).
#pragma once

#include "pairs.cuh"

namespace so3lr_b200 {

constexpr float kInvSqrt2Pi = 0.39894228f;
constexpr float kTanhSlope = 1.5957691f, kTanhCube = 0.044715f;  // 2 sqrt(2 / pi)

template <int ACT>
__device__ __forceinline__ Pair activate(const Pair &z);
// gelu: z Phi(z), see normal_cdf.
// gelu_tanh: z (1 + tanh(u)) / 2 = z sigmoid(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3). relu keeps a NaN.
template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if (ACT == SO3LR_RELU) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(z) : "f"(0.0f));
    return z;
  }
  if (ACT == SO3LR_NO_ACTIVATION) return z;
  float a, b;
  activate<ACT>(Pair(z)).get(a, b);
  return a;
}
// The derivative at a finite z or a NaN; beyond 1000 the s (1 - s) of gelu_tanh is 0, and the
// square would become infinite.
template <int ACT>
__device__ __forceinline__ float slope(float z) {
  return ACT == SO3LR_RELU ? (z > 0.0f ? 1.0f : z <= 0.0f ? 0.0f : z) : 1.0f;
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
// The same of pairs: what is not a function of the hardware takes one instruction for both.
__device__ __forceinline__ Pair sigmoid_pair(const Pair &negative_log2) {  // 1 / (1 + 2^v)
  float a, b;
  negative_log2.get(a, b);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
  (Pair(a, b) + Pair(1.0f)).get(a, b);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
  return Pair(a, b);
}
constexpr float kLog2E = 1.4426950408889634f;
__device__ __forceinline__ Pair tanh_sigmoid(const Pair &z) {  // sigmoid(2 u) of gelu_tanh
  const Pair cube = z * Pair(kTanhCube) * z;
  return sigmoid_pair(madd(cube, z, z) * Pair(-kTanhSlope * kLog2E));
}
// Phi(z) and e = exp(-z^2 / 2). Phi(-|z|) = t poly(t) e with t = 1 / (1 + 0.35 |z|), the form of
// Hastings' approximations of erf. The coefficients were fitted here (a linear program over 6000 points of
// |z| <= 14) so that the largest of the relative error / 5e-6 and the absolute error / 3e-8 is least, 1.04: far
// out, where z Phi(z) is small, it keeps its leading digits too. In float32 arithmetic 2e-7 and, up to |z| = 12,
// 2e-5 of the value. (Abramowitz and Stegun's 7.1.26, of two terms fewer, is off by 1 % at z = -8 for the same
// absolute error.)
__device__ __forceinline__ Pair normal_cdf(const Pair &z, Pair &e) {
  float a, b, ta, tb, ea, eb;
  z.get(a, b);
  madd(Pair(fabsf(a), fabsf(b)), Pair(0.35f), Pair(1.0f)).get(ta, tb);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(ta));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(tb));
  (z * z * Pair(-0.5f * kLog2E)).get(ea, eb);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(ea));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(eb));
  const Pair t(ta, tb);
  e = Pair(ea, eb);
  Pair q = madd(t, Pair(0.0441702157f), Pair(-0.182627589f));
  q = madd(q, t, Pair(0.208162174f));
  q = madd(q, t, Pair(0.0113299619f));
  q = madd(q, t, Pair(0.142112911f));
  q = madd(q, t, Pair(0.137093723f));
  q = madd(q, t, Pair(0.139758632f)) * (t * e);
  float qa, qb;
  q.get(qa, qb);
  return Pair(a < 0.0f ? qa : 1.0f - qa, b < 0.0f ? qb : 1.0f - qb);
}
template <int ACT>
__device__ __forceinline__ Pair activate(const Pair &z) {
  if (ACT == SO3LR_SILU) return z * sigmoid_pair(z * Pair(-kLog2E));
  if (ACT == SO3LR_GELU) {
    Pair e;
    return z * normal_cdf(z, e);
  }
  if (ACT == SO3LR_GELU_TANH) return z * tanh_sigmoid(z);
  if (ACT == SO3LR_RELU) {
    float a, b;
    z.get(a, b);
    return Pair(activate<ACT>(a), activate<ACT>(b));
  }
  return z;
}
template <int ACT>
__device__ __forceinline__ Pair slope(const Pair &z) {
  if (ACT == SO3LR_SILU) {
    const Pair s = sigmoid_pair(z * Pair(-kLog2E));
    return s * madd(z, madd(s, Pair(-1.0f), Pair(1.0f)), Pair(1.0f));
  }
  if (ACT == SO3LR_GELU) {
    Pair e;
    const Pair cdf = normal_cdf(z, e);
    return madd(z * Pair(kInvSqrt2Pi), e, cdf);
  }
  float a, b;
  z.get(a, b);
  if (ACT == SO3LR_GELU_TANH) {
    const Pair s = tanh_sigmoid(z), c(fminf(fmaxf(a, -1000.0f), 1000.0f), fminf(fmaxf(b, -1000.0f), 1000.0f));
    const Pair rise = c * Pair(kTanhSlope) * madd(c * Pair(3.0f * kTanhCube), c, Pair(1.0f));
    return madd(rise, s * madd(s, Pair(-1.0f), Pair(1.0f)), s);
  }
  if (ACT == SO3LR_RELU) return Pair(slope<ACT>(a), slope<ACT>(b));
  return Pair(1.0f);
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
