// AdamW over many tensors at once, moments in 32 bits or in 8.
//
//   m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr decay) - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)
//
// Bound by HBM: an element is read and written once (28 bytes with 32-bit moments, 16
// with 8-bit ones and a float32 master). Every tensor is cut into chunks of 2048
// elements, a chunk is a block's work, and one launch covers all tensors: a block finds
// its tensor in a table that travels as the kernel's argument, so that nothing is
// copied to the GPU before it and a captured graph holds its own table. The step
// counters live on the GPU: a first small kernel adds one to each and works out its
// bias corrections in float64, where 1 - beta^t keeps its digits for small t.
//
// An 8-bit moment is a code for each element and, for each 256 of them, the largest
// magnitude `top`: m = top t |t| with t = code / 127, v = top t^4 with t = code / 255.
// The roots spread the codes over the magnitudes that a block mixes: m down to 6e-5 of
// the largest, the root of v to 1.5e-5, both with steps of at most 1.6 % (v: 1.6 %) near
// the largest, and the largest itself is kept exactly, so that a block decays as its
// moments do. Codes are rounded to nearest. A v that is not zero never becomes zero
// (its code is 1 at least): m / sqrt(v) would otherwise run away. One warp holds the 256
// elements of a scale, eight to a lane.
#include <algorithm>

#include "adamw.hpp"
#include "layers_common.cuh"

namespace so3lr_b200 {
namespace {

constexpr int kChunk = 2048, kScaleBlock = 256, kPer = 8, kAdamThreads = kChunk / kPer;

struct Entry {
  void *p;
  const void *g;
  float *master;       // nullptr: p is what is updated
  void *m, *v;         // float, or codes where the scales are given
  float *m_top, *v_top;
  long long n;
};
// What a block needs to know of a tensor's types
enum Kind : unsigned char { kParamMask = 3, kGradFloat = 4, kEight = 8, kWide = 16 };

template <int MOST>
struct Table {
  Entry e[MOST];
  int first[MOST + 1];  // first chunk of each tensor, and their number
  unsigned char kind[MOST];
  int count;
  const float4 *coef;   // of the first tensor: lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), 1 - lr decay
  float b1, c1, b2, c2, eps;
};
template <int MOST>
struct Steps {
  long long *step[MOST];
  int count;
  float4 *coef;
  double lr;
  const float *lr_device;
  double beta1, beta2, decay;
};

template <int MOST>
__global__ void k_adamw_steps(const __grid_constant__ Steps<MOST> a) {
  dependents_may_start();
  wait_for_predecessors();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.count) return;
  const long long t = *a.step[i] + 1;
  *a.step[i] = t;
  const double lr = a.lr_device ? double(*a.lr_device) : a.lr;
  a.coef[i] = make_float4(float(lr / (1.0 - pow(a.beta1, double(t)))), float(1.0 / sqrt(1.0 - pow(a.beta2, double(t)))),
                          float(1.0 - lr * a.decay), 0.0f);
}

// kPer consecutive elements as float, or `left` of them one by one
template <class T>
__device__ __forceinline__ void read(const T *p, bool whole, int left, float (&f)[kPer]) {
  if (whole) {
    const Chunk<T, kPer> c = load_chunk<T, kPer>(p);
#pragma unroll
    for (int i = 0; i < kPer; ++i) f[i] = to_float(c.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) f[i] = i < left ? to_float(p[i]) : 0.0f;
  }
}
template <class T>
__device__ __forceinline__ void write(T *p, bool whole, int left, const float (&f)[kPer]) {
  const Chunk<T, kPer> c = to_chunk<T, kPer>(f);
  if (whole) {
    store_chunk<T, kPer>(p, c);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < left) p[i] = c.e[i];
  }
}
using Codes = Chunk<unsigned char, kPer>;
__device__ __forceinline__ Codes read_codes(const void *p, bool whole, int left) {
  if (whole) return load_chunk<unsigned char, kPer>(static_cast<const unsigned char *>(p));
  Codes c{};
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (i < left) c.e[i] = static_cast<const unsigned char *>(p)[i];
  return c;
}
__device__ __forceinline__ void write_codes(void *p, bool whole, int left, const Codes &c) {
  if (whole) return store_chunk<unsigned char, kPer>(static_cast<unsigned char *>(p), c);
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (i < left) static_cast<unsigned char *>(p)[i] = c.e[i];
}

// What a code stands for. SIGNED: m, else v.
template <bool SIGNED>
__device__ __forceinline__ float value_of(unsigned char code, float top) {
  if (SIGNED) {
    const float t = float(static_cast<signed char>(code)) * (1.0f / 127.0f);
    return t * fabsf(t) * top;
  }
  const float t = float(code) * (1.0f / 255.0f), square = t * t;
  return square * square * top;
}
__device__ __forceinline__ float root(float v) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// The warp's 256 elements to codes; returns their scale. A block that holds an infinity
// or a NaN gets scale NaN and codes 0, one whose largest is below float32's normal
// numbers (its reciprocal could overflow) scale 0 and codes 0.
template <bool SIGNED>
__device__ __forceinline__ float encode(const float (&f)[kPer], Codes &codes) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) top = max_abs(top, f[i]);
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top) & 0x7fffffffu);
  top = __uint_as_float(bits);
  if (bits > 0x7f7fffffu || bits < 0x00800000u) {
    codes = Codes{};
    return bits > 0x7f7fffffu ? __uint_as_float(0x7fc00000u) : 0.0f;
  }
  const float inv = 1.0f / top;
  // adding 1.5 2^23 leaves the rounded integer in the low bits of the sum
  uint32_t q[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (SIGNED) {
      q[i] = __float_as_uint(fmaf(copysignf(root(fabsf(f[i]) * inv), f[i]), 127.0f, 12582912.0f));
    } else {
      const float code = root(root(f[i] * inv)) * 255.0f;
      q[i] = __float_as_uint((f[i] > 0.0f ? fmaxf(code, 1.0f) : 0.0f) + 12582912.0f);
    }
  }
#pragma unroll
  for (int i = 0; i < kPer / 4; ++i) {
    const uint32_t lo = __byte_perm(q[4 * i], q[4 * i + 1], 0x0040), hi = __byte_perm(q[4 * i + 2], q[4 * i + 3], 0x0040);
    reinterpret_cast<uint32_t *>(&codes)[i] = __byte_perm(lo, hi, 0x5410);
  }
  return top;
}

template <class P, class G, bool EIGHT, int MOST>
__device__ __forceinline__ void update(const Table<MOST> &a, const Entry &e, bool wide, long long chunk, const float4 &coef) {
  const long long at = chunk * kChunk + threadIdx.x * kPer;
  const int left = int(min((long long)kPer, e.n - at));  // may be negative; a warp past the end has nothing to do
  const bool whole = wide && left == kPer;
  if (at - (threadIdx.x & 31) * kPer >= e.n) return;
  float g[kPer], p[kPer], m[kPer], v[kPer];
  read(static_cast<const G *>(e.g) + at, whole, left, g);
  if (e.master)
    read(e.master + at, whole, left, p);
  else
    read(static_cast<const P *>(e.p) + at, whole, left, p);
  const long long block = at / kScaleBlock;
  if (EIGHT) {
    const Codes cm = read_codes(static_cast<unsigned char *>(e.m) + at, whole, left);
    const Codes cv = read_codes(static_cast<unsigned char *>(e.v) + at, whole, left);
    const float m_top = e.m_top[block], v_top = e.v_top[block];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      m[i] = value_of<true>(cm.e[i], m_top);
      v[i] = value_of<false>(cv.e[i], v_top);
    }
  } else {
    read(static_cast<const float *>(e.m) + at, whole, left, m);
    read(static_cast<const float *>(e.v) + at, whole, left, v);
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    m[i] = fmaf(a.b1, m[i], a.c1 * g[i]);
    v[i] = fmaf(a.b2, v[i], a.c2 * (g[i] * g[i]));
    // the denominator is at least eps and far below 2^126, where the fast division is exact to 2 units
    p[i] = fmaf(p[i], coef.z, -coef.x * __fdividef(m[i], fmaf(root(v[i]), coef.y, a.eps)));
  }
  if (EIGHT) {
    if (left < kPer) {  // what is behind the end does not count in the scale
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i >= left) m[i] = v[i] = 0.0f;
    }
    Codes cm, cv;
    const float m_top = encode<true>(m, cm), v_top = encode<false>(v, cv);
    write_codes(static_cast<unsigned char *>(e.m) + at, whole, left, cm);
    write_codes(static_cast<unsigned char *>(e.v) + at, whole, left, cv);
    if ((threadIdx.x & 31) == 0) {
      e.m_top[block] = m_top;
      e.v_top[block] = v_top;
    }
  } else {
    write(static_cast<float *>(e.m) + at, whole, left, m);
    write(static_cast<float *>(e.v) + at, whole, left, v);
  }
  if (e.master) write(e.master + at, whole, left, p);
  write(static_cast<P *>(e.p) + at, whole, left, p);
}

template <int MOST>
__global__ void __launch_bounds__(kAdamThreads) k_adamw(const __grid_constant__ Table<MOST> a) {
  dependents_may_start();
  int lo = 0, hi = a.count - 1;  // the last tensor whose first chunk is not behind this block's
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (a.first[mid] <= int(blockIdx.x))
      lo = mid;
    else
      hi = mid - 1;
  }
  const Entry &e = a.e[lo];
  const int kind = a.kind[lo];
  const long long chunk = blockIdx.x - a.first[lo];
  const bool wide = kind & kWide;
  wait_for_predecessors();
  const float4 coef = a.coef[lo];
  switch (kind & (kParamMask | kGradFloat | kEight)) {
    case SO3LR_FLOAT32 | kGradFloat: return update<float, float, false>(a, e, wide, chunk, coef);
    case SO3LR_FLOAT32 | kGradFloat | kEight: return update<float, float, true>(a, e, wide, chunk, coef);
    case SO3LR_BFLOAT16: return update<__nv_bfloat16, __nv_bfloat16, false>(a, e, wide, chunk, coef);
    case SO3LR_BFLOAT16 | kEight: return update<__nv_bfloat16, __nv_bfloat16, true>(a, e, wide, chunk, coef);
    case SO3LR_BFLOAT16 | kGradFloat: return update<__nv_bfloat16, float, false>(a, e, wide, chunk, coef);
    case SO3LR_BFLOAT16 | kGradFloat | kEight: return update<__nv_bfloat16, float, true>(a, e, wide, chunk, coef);
    case SO3LR_FLOAT16: return update<__half, __half, false>(a, e, wide, chunk, coef);
    case SO3LR_FLOAT16 | kEight: return update<__half, __half, true>(a, e, wide, chunk, coef);
    case SO3LR_FLOAT16 | kGradFloat: return update<__half, float, false>(a, e, wide, chunk, coef);
    case SO3LR_FLOAT16 | kGradFloat | kEight: return update<__half, float, true>(a, e, wide, chunk, coef);
  }
}

// values = what an 8-bit moment's codes stand for
template <class O, bool SIGNED>
__global__ void k_moment_values(const so3lr_moment_values_args a, bool wide) {
  dependents_may_start();
  wait_for_predecessors();
  const unsigned char *codes = static_cast<const unsigned char *>(a.codes);
  for (long long at = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * kPer; at < a.n;
       at += (long long)gridDim.x * blockDim.x * kPer) {
    const int left = int(min((long long)kPer, a.n - at));
    const bool whole = wide && left == kPer;
    const Codes c = read_codes(codes + at, whole, left);
    const float top = a.scales[at / kScaleBlock];
    float f[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) f[i] = value_of<SIGNED>(c.e[i], top);
    write(static_cast<O *>(a.values) + at, whole, left, f);
  }
}

bool on(const void *p, std::size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <int MOST>
void launch_step(const so3lr_adamw_args &a, float4 *coef, cudaStream_t s) {
  for (long long begin = 0; begin < a.count; begin += MOST) {
    Steps<MOST> steps{};
    steps.count = int(std::min<long long>(MOST, a.count - begin));
    steps.coef = coef + begin;
    steps.lr = a.lr;
    steps.lr_device = a.lr_device;
    steps.beta1 = a.beta1;
    steps.beta2 = a.beta2;
    steps.decay = a.weight_decay;
    for (int i = 0; i < steps.count; ++i) steps.step[i] = a.tensors[begin + i].step;
    launch(k_adamw_steps<MOST>, unsigned((steps.count + 31) / 32), 32, 0, s, steps);
  }
  Table<MOST> t{};
  t.b1 = float(a.beta1);
  t.c1 = float(1.0 - a.beta1);
  t.b2 = float(a.beta2);
  t.c2 = float(1.0 - a.beta2);
  t.eps = float(a.eps);
  auto flush = [&] {
    if (t.count && t.first[t.count]) launch(k_adamw<MOST>, unsigned(t.first[t.count]), kAdamThreads, 0, s, t);
    t.count = 0;
  };
  for (long long i = 0; i < a.count; ++i) {
    const so3lr_adamw_tensor &x = a.tensors[i];
    const long long chunks = (x.n + kChunk - 1) / kChunk;  // 2^30 at most
    if (t.count == MOST || (t.count && t.first[t.count] + chunks > 0x7fffffffLL)) flush();
    if (t.count == 0) t.coef = coef + i;
    t.e[t.count] = Entry{x.param, x.grad, x.master, x.exp_avg, x.exp_avg_sq, x.exp_avg_scale, x.exp_avg_sq_scale, x.n};
    const std::size_t e = x.dtype == SO3LR_FLOAT32 ? 4 : 2, ge = x.grad_dtype == SO3LR_FLOAT32 ? 4 : 2;
    const std::size_t moment = x.exp_avg_scale ? 8 : 16;
    const bool wide = on(x.param, std::min<std::size_t>(16, e * kPer)) && on(x.grad, std::min<std::size_t>(16, ge * kPer)) &&
                      on(x.master, 16) && on(x.exp_avg, moment) && on(x.exp_avg_sq, moment);
    t.kind[t.count] = static_cast<unsigned char>(x.dtype | (x.grad_dtype == SO3LR_FLOAT32 ? kGradFloat : 0) |
                                                 (x.exp_avg_scale ? kEight : 0) | (wide ? kWide : 0));
    t.first[t.count + 1] = int(t.first[t.count] + chunks);
    ++t.count;
  }
  flush();
}

}  // namespace

long long adamw_bytes(const so3lr_adamw_args &a) { return a.count * (long long)sizeof(float4); }

// A table of 24 tensors (1.8 KB of arguments) where they fit: the driver copies the
// whole argument at every launch, 28 KB for 400 tensors.
void launch_adamw(const so3lr_adamw_args &a, void *workspace, cudaStream_t s) {
  float4 *coef = static_cast<float4 *>(workspace);
  if (a.count <= 24)
    launch_step<24>(a, coef, s);
  else
    launch_step<400>(a, coef, s);
}

void launch_moment_values(const so3lr_moment_values_args &a, cudaStream_t s) {
  const bool wide = on(a.codes, 8) && on(a.values, 16);
  const unsigned grid = unsigned(std::min<long long>((a.n + 256 * kPer - 1) / (256 * kPer), kSmCount * 32));
  auto go = [&](auto t) {
    using O = decltype(t);
    launch(a.is_signed ? &k_moment_values<O, true> : &k_moment_values<O, false>, grid, 256, 0, s, a, wide);
  };
  if (a.dtype == SO3LR_FLOAT32)
    go(float{});
  else if (a.dtype == SO3LR_BFLOAT16)
    go(__nv_bfloat16{});
  else
    go(__half{});
}

}  // namespace so3lr_b200
