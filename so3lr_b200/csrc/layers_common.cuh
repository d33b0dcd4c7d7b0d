// Element types, vector chunks and row reductions of the row-wise feed-forward
// layers (rows.cu, dense*.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "layers.hpp"

namespace so3lr_b200 {

constexpr int kSmCount = 148;  // B200

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// VEC consecutive elements, moved in pieces of at most 16 bytes. VEC > 1 needs the
// address aligned to min(16, VEC * sizeof(T)).
template <class T, int VEC>
struct alignas(VEC * sizeof(T) < 16 ? VEC * sizeof(T) : 16) Chunk {
  T e[VEC];
};
template <class T, int VEC>
__device__ __forceinline__ Chunk<T, VEC> load_chunk(const T *p) {
  return *reinterpret_cast<const Chunk<T, VEC> *>(p);
}
template <class T, int VEC>
__device__ __forceinline__ void store_chunk(T *p, const Chunk<T, VEC> &c) {
  *reinterpret_cast<Chunk<T, VEC> *>(p) = c;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// silu(g) = g / (1 + exp(-g)). exp(-g) overflows to infinity for g < -88 and the
// quotient is then 0, as it should be to float32's range.
__device__ __forceinline__ float silu_f32(float g) { return __fdividef(g, 1.0f + __expf(-g)); }

// max|v| of a row from the bits of |v|, which order like the values with
// infinities and NaN on top. Row scale: 0 for a row whose scale would not be a
// normal number (its reciprocal could overflow), NaN for one that holds an
// infinity or a NaN; `inv` is then 0, which makes every code 0.
__device__ __forceinline__ float row_scale(uint32_t top_bits, float &inv) {
  inv = 0.0f;
  if (top_bits > 0x7f7fffffu) return __uint_as_float(0x7fc00000u);
  const float scale = __uint_as_float(top_bits) / 127.0f;
  if (scale < 1.17549435e-38f) return 0.0f;
  inv = 1.0f / scale;
  return scale;
}
__device__ __forceinline__ signed char to_code(float v, float inv) {
  // a NaN can only meet inv = 0 here; __float2int_rn turns the NaN product into 0
  return static_cast<signed char>(max(-127, min(127, __float2int_rn(v * inv))));
}

}  // namespace so3lr_b200
