// Element types, vector chunks and row reductions of the row-wise feed-forward
// layers (rows.cu, dense*.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>
#include <utility>

#include "layers.hpp"

namespace so3lr_b200 {

constexpr int kSmCount = 148;  // B200

// Programmatic dependent launch. Every kernel of the layers is launched so that it may
// start while the kernel before it on the stream finishes: it lets its own successor
// start (dependents_may_start) and touches no global memory before
// wait_for_predecessors, which returns when everything before it on the stream has
// completed and is visible. What runs ahead is launch latency and set-up (barriers,
// TMEM, tensor maps), 1 to 2 us of a small call's kernels.
__device__ __forceinline__ void dependents_may_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_for_predecessors() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <class... P, class... A>
void launch_clusters(void (*kernel)(P...), dim3 grid, dim3 block, unsigned cluster, std::size_t smem,
                     cudaStream_t stream, A &&...args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = attr;
  config.numAttrs = cluster ? 2 : 1;  // 0: as the kernel declares
  ++launch_counter();
  SO3_CUDA(cudaLaunchKernelEx(&config, kernel, std::forward<A>(args)...));
}
template <class... P, class... A>
void launch(void (*kernel)(P...), dim3 grid, dim3 block, std::size_t smem, cudaStream_t stream, A &&...args) {
  launch_clusters(kernel, grid, block, 0, smem, stream, std::forward<A>(args)...);
}

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

// VEC values rounded to T. Pairs go through one packed conversion: element by element
// it is a conversion and a byte permutation each.
template <class T, int VEC>
__device__ __forceinline__ Chunk<T, VEC> to_chunk(const float (&v)[VEC]) {
  Chunk<T, VEC> c;
  if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      if constexpr (std::is_same<T, __half>::value)
        *reinterpret_cast<__half2 *>(&c.e[i]) = __floats2half2_rn(v[i], v[i + 1]);
      else
        *reinterpret_cast<__nv_bfloat162 *>(&c.e[i]) = __floats2bfloat162_rn(v[i], v[i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) c.e[i] = from_float<T>(v[i]);
  }
  return c;
}

// 1 / (1 + exp(-g)) with the hardware's exponential and reciprocal, within 2 units in the
// last place each, besides the rounding of the exponential's argument: up to 0.6 |g| units
// of exp(-g), which show where it is not small beside 1 (g = -10: 6 units of a sigmoid of
// 4e-5; g = -80: 50 of one of 2e-35). exp(-g) overflows to infinity for g < -88, and the
// result is then 0, as it should be to float32's range; the flushed denormals of either do
// not show beside 1.
__device__ __forceinline__ float sigmoid_f32(float g) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}
__device__ __forceinline__ float silu_f32(float g) { return g * sigmoid_f32(g); }

// |result| = max(|a|, |b|), a NaN if either is one (the sign is the product of
// theirs): one instruction per element of a row's maximum
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Row scale from the bits of max|v|, which order like the values with infinities
// and NaN on top: 0 for a row whose scale would not be a normal number (its
// reciprocal could overflow), NaN for one that holds an infinity or a NaN. `inv` is
// then 0, which makes every code 0.
__device__ __forceinline__ float row_scale(uint32_t top_bits, float &inv) {
  inv = 0.0f;
  if (top_bits > 0x7f7fffffu) return __uint_as_float(0x7fc00000u);
  const float scale = __uint_as_float(top_bits) * (1.0f / 127.0f);
  if (scale < 1.17549435e-38f) return 0.0f;
  inv = __fdividef(1.0f, scale);
  return scale;
}
// VEC codes of a row: v inv rounded to nearest even. Adding 1.5 2^23 leaves the
// rounded integer in the low bits of the sum (a float-to-int conversion runs at an
// eighth of the rate); |v inv| <= 127 (1 + 2^-22), so the low byte is the code.
template <int VEC>
__device__ __forceinline__ Chunk<signed char, VEC> to_codes(const float *v, float inv) {
  Chunk<signed char, VEC> out;
  uint32_t q[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) q[i] = __float_as_uint(fmaf(v[i], inv, 12582912.0f));
  if (VEC % 4 == 0) {
    const uint32_t live = inv != 0.0f ? 0xffffffffu : 0u;
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const uint32_t lo = __byte_perm(q[4 * i], q[4 * i + 1], 0x0040);
      const uint32_t hi = __byte_perm(q[4 * i + 2], q[4 * i + 3], 0x0040);
      reinterpret_cast<uint32_t *>(&out)[i] = __byte_perm(lo, hi, 0x5410) & live;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) out.e[i] = inv != 0.0f ? static_cast<signed char>(q[i] & 0xff) : 0;
  }
  return out;
}
// The float of a signed byte, without the slow int-to-float conversion: the byte
// + 128 in the low bits of 2^23
__device__ __forceinline__ float byte_to_float(uint32_t flipped, int i) {
  return __uint_as_float(__byte_perm(flipped, 0x4b000000u, 0x7440 + i)) - 8388736.0f;
}

}  // namespace so3lr_b200
