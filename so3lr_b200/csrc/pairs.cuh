// Two floats in one register pair: their products, sums and multiply-adds issue as one
// instruction, each half rounded by itself. And elements of rows as such pairs.
#pragma once

#include "layers_common.cuh"

namespace so3lr_b200 {

struct Pair {
  uint64_t bits;
  Pair() = default;
  __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(a), "f"(b)); }
  __device__ __forceinline__ explicit Pair(float a) : Pair(a, a) {}
  __device__ __forceinline__ Pair(uint64_t b, int) : bits(b) {}
  __device__ __forceinline__ void get(float &a, float &b) const {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(bits));
  }
};
__device__ __forceinline__ Pair operator*(const Pair &a, const Pair &b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a.bits), "l"(b.bits));
  return Pair(r, 0);
}
// The assembler contracts a sum with a product that it adds.
__device__ __forceinline__ Pair operator+(const Pair &a, const Pair &b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a.bits), "l"(b.bits));
  return Pair(r, 0);
}
// a b + c, of pairs or of floats
__device__ __forceinline__ Pair madd(const Pair &a, const Pair &b, const Pair &c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
  return Pair(r, 0);
}
__device__ __forceinline__ float madd(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float total(const Pair &v) {
  float a, b;
  v.get(a, b);
  return a + b;
}
__device__ __forceinline__ float total(float v) { return v; }

// VEC elements of a row as floats: in pairs where there are two.
template <int VEC>
struct Floats {
  using V = typename std::conditional<(VEC > 1), Pair, float>::type;
  static constexpr int kCount = VEC > 1 ? VEC / 2 : 1;
  V v[kCount];
};
// From a chunk by whole words: a bfloat16 is the upper half of its float.
template <class T, int VEC>
__device__ __forceinline__ Floats<VEC> floats_of(const Chunk<T, VEC> &c) {
  Floats<VEC> f;
  if constexpr (VEC == 1) {
    f.v[0] = to_float(c.e[0]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const uint32_t w = reinterpret_cast<const uint32_t *>(&c)[i];
        f.v[i] = Pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 p = __half22float2(reinterpret_cast<const __half2 *>(&c)[i]);
        f.v[i] = Pair(p.x, p.y);
      } else {
        f.v[i] = Pair(c.e[2 * i], c.e[2 * i + 1]);
      }
    }
  }
  return f;
}
template <class T, int VEC>
__device__ __forceinline__ Chunk<T, VEC> chunk_of_floats(const Floats<VEC> &f) {
  float v[VEC];
  if constexpr (VEC == 1) {
    v[0] = f.v[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) f.v[i].get(v[2 * i], v[2 * i + 1]);
  }
  return to_chunk<T, VEC>(v);
}
// a chunk of ones, for a factor that is not there
template <class T, int VEC>
__device__ __forceinline__ Chunk<T, VEC> ones() {
  Chunk<T, VEC> c;
#pragma unroll
  for (int i = 0; i < VEC; ++i) c.e[i] = from_float<T>(1.0f);
  return c;
}

}  // namespace so3lr_b200
