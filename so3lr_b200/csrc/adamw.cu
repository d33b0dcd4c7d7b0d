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

// kPer consecutive elements as float; not WHOLE: the `left` first of them one by one, zeros for the others
template <bool WHOLE, class T>
__device__ __forceinline__ void read(const T *p, int left, float (&f)[kPer]) {
  if (WHOLE) {
    const Chunk<T, kPer> c = load_chunk<T, kPer>(p);
#pragma unroll
    for (int i = 0; i < kPer; ++i) f[i] = to_float(c.e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) f[i] = i < left ? to_float(p[i]) : 0.0f;
  }
}
template <bool WHOLE, class T>
__device__ __forceinline__ void write(T *p, int left, const float (&f)[kPer]) {
  const Chunk<T, kPer> c = to_chunk<T, kPer>(f);
  if (WHOLE) {
    store_chunk<T, kPer>(p, c);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < left) p[i] = c.e[i];
  }
}
// kPer codes, in words: bytes by themselves would take a register and an instruction each
struct Codes {
  uint32_t word[kPer / 4];
};
template <bool WHOLE>
__device__ __forceinline__ Codes read_codes(const void *from, int left) {
  const unsigned char *p = static_cast<const unsigned char *>(from);
  Codes c{};
  if (WHOLE) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    c.word[0] = v.x;
    c.word[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < left) c.word[i / 4] |= uint32_t(p[i]) << 8 * (i % 4);
  }
  return c;
}
template <bool WHOLE>
__device__ __forceinline__ void write_codes(void *to, int left, const Codes &c) {
  unsigned char *p = static_cast<unsigned char *>(to);
  if (WHOLE) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(c.word[0], c.word[1]);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < left) p[i] = static_cast<unsigned char>(c.word[i / 4] >> 8 * (i % 4));
  }
}

// What a code stands for. SIGNED: m, else v. Each product is rounded by itself: what a state
// stands for must not depend on how a compiler contracts.
__device__ __forceinline__ float of_m(float code, float top) {
  const float t = __fmul_rn(code, 1.0f / 127.0f);
  return __fmul_rn(__fmul_rn(t, fabsf(t)), top);
}
__device__ __forceinline__ float of_v(float code, float top) {
  const float t = __fmul_rn(code, 1.0f / 255.0f), square = __fmul_rn(t, t);
  return __fmul_rn(__fmul_rn(square, square), top);
}
// kPer values of codes, without the slow int-to-float conversion: a byte in the low bits of 2^23
template <bool SIGNED>
__device__ __forceinline__ void values_of(const Codes &codes, float top, float (&f)[kPer]) {
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t word = codes.word[i / 4];
    if (SIGNED)
      f[i] = of_m(byte_to_float(word ^ 0x80808080u, i % 4), top);
    else
      f[i] = of_v(__uint_as_float(__byte_perm(word, 0x4b000000u, 0x7440 + i % 4)) - 8388608.0f, top);
  }
}
__device__ __forceinline__ float root(float v) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// The square root of x in 2^-126..1 as correctly rounded (but for one in a million, which is a
// unit off): Heron's step on x times the hardware's reciprocal root. With the approximate
// root alone one code in 30,000 would fall on the other side of a tie.
__device__ __forceinline__ float root_of_share(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  const float s = x * y;
  return fmaf(fmaf(-s, s, x), 0.5f * y, s);
}
// The largest magnitude of the warp's 256 elements, for a scale; `live`: codes can be made
// with it. Not of a block that holds an infinity or a NaN (scale NaN, codes 0), nor of one
// whose largest is below float32's normal numbers (scale 0, codes 0: its reciprocal could
// overflow).
__device__ __forceinline__ float scale_of(const float (&f)[kPer], bool &live) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) top = max_abs(top, f[i]);
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top) & 0x7fffffffu);
  live = bits <= 0x7f7fffffu && bits >= 0x00800000u;
  return live ? __uint_as_float(bits) : bits > 0x7f7fffffu ? __uint_as_float(0x7fc00000u) : 0.0f;
}
// The shares of the scale, 2^-126 at least: smaller ones get code 0 (or 1) either way.
__device__ __forceinline__ float share_of(float f, float inv) { return fmaxf(fabsf(f) * inv, 0x1p-126f); }
// Codes from their values: adding 1.5 2^23 leaves the rounded integer in the low bits of the sum.
__device__ __forceinline__ Codes pack(const float (&code)[kPer]) {
  Codes codes;
  uint32_t q[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) q[i] = __float_as_uint(__fadd_rn(code[i], 12582912.0f));
#pragma unroll
  for (int i = 0; i < kPer / 4; ++i) {
    const uint32_t lo = __byte_perm(q[4 * i], q[4 * i + 1], 0x0040), hi = __byte_perm(q[4 * i + 2], q[4 * i + 3], 0x0040);
    codes.word[i] = __byte_perm(lo, hi, 0x5410);
  }
  return codes;
}
__device__ __forceinline__ float reciprocal(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// What of a tensor a block needs, and the coefficients of its step
struct Work {
  const Entry &e;
  float4 coef;
  float b1, c1, b2, c2, eps;
};
// WHOLE: all of the warp's elements are there and on 16-byte boundaries
template <class P, class G, bool EIGHT, bool WHOLE>
__device__ __forceinline__ void update(const Work &a, long long at) {
  const Entry &e = a.e;
  const float4 coef = a.coef;
  const int left = WHOLE ? kPer : int(min((long long)kPer, e.n - at));  // may be negative
  float g[kPer], p[kPer], m[kPer], v[kPer];
  read<WHOLE>(static_cast<const G *>(e.g) + at, left, g);
  if (e.master)
    read<WHOLE>(e.master + at, left, p);
  else
    read<WHOLE>(static_cast<const P *>(e.p) + at, left, p);
  const long long block = at / kScaleBlock;
  if (EIGHT) {
    const Codes cm = read_codes<WHOLE>(static_cast<unsigned char *>(e.m) + at, left);
    const Codes cv = read_codes<WHOLE>(static_cast<unsigned char *>(e.v) + at, left);
    // what is behind the end stays zero, and so does not count in the scale
    values_of<true>(cm, e.m_top[block], m);
    values_of<false>(cv, e.v_top[block], v);
  } else {
    read<WHOLE>(static_cast<const float *>(e.m) + at, left, m);
    read<WHOLE>(static_cast<const float *>(e.v) + at, left, v);
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    m[i] = __fadd_rn(__fmul_rn(a.b1, m[i]), __fmul_rn(a.c1, g[i]));
    v[i] = __fadd_rn(__fmul_rn(a.b2, v[i]), __fmul_rn(a.c2, __fmul_rn(g[i], g[i])));
  }
  // the denominator is at least eps, a normal number, and below 2^126
  auto move = [&](int i, float denominator) { p[i] = fmaf(p[i], coef.z, -coef.x * (m[i] * reciprocal(denominator))); };
  if (EIGHT) {
    bool m_live, v_live;
    const float m_top = scale_of(m, m_live), v_top = scale_of(v, v_live);
    float code[kPer];
    Codes cm{}, cv{};
    if (v_live) {  // the root of v is that of its share, which its code needs too
      const float inv = __frcp_rn(v_top), back = root(v_top) * coef.y;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const float half = root_of_share(share_of(v[i], inv));
        move(i, fmaf(half, back, a.eps));
        code[i] = __fmul_rn(root_of_share(half), 255.0f);
        if (v[i] > 0.0f) code[i] = fmaxf(code[i], 1.0f);
      }
      cv = pack(code);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) move(i, fmaf(root(v[i]), coef.y, a.eps));
    }
    if (m_live) {
      const float inv = __frcp_rn(m_top);
#pragma unroll
      for (int i = 0; i < kPer; ++i) code[i] = copysignf(__fmul_rn(root_of_share(share_of(m[i], inv)), 127.0f), m[i]);
      cm = pack(code);
    }
    write_codes<WHOLE>(static_cast<unsigned char *>(e.m) + at, left, cm);
    write_codes<WHOLE>(static_cast<unsigned char *>(e.v) + at, left, cv);
    if ((threadIdx.x & 31) == 0) {
      e.m_top[block] = m_top;
      e.v_top[block] = v_top;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) move(i, fmaf(root(v[i]), coef.y, a.eps));
    write<WHOLE>(static_cast<float *>(e.m) + at, left, m);
    write<WHOLE>(static_cast<float *>(e.v) + at, left, v);
  }
  if (e.master) write<WHOLE>(e.master + at, left, p);
  write<WHOLE>(static_cast<P *>(e.p) + at, left, p);
}

template <class P, class G, bool EIGHT>
__device__ __forceinline__ void update_chunk(const Work &a, long long chunk, bool wide) {
  const long long at = chunk * kChunk + threadIdx.x * kPer, warp_at = at - (threadIdx.x & 31) * kPer;
  if (wide && warp_at + 32 * kPer <= a.e.n)
    update<P, G, EIGHT, true>(a, at);
  else if (warp_at < a.e.n)
    update<P, G, EIGHT, false>(a, at);
}

template <int MOST>
__global__ void __launch_bounds__(kAdamThreads) k_adamw(const __grid_constant__ Table<MOST> t) {
  dependents_may_start();
  int lo = 0, hi = t.count - 1;  // the last tensor whose first chunk is not behind this block's
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.first[mid] <= int(blockIdx.x))
      lo = mid;
    else
      hi = mid - 1;
  }
  const int kind = t.kind[lo];
  const long long chunk = blockIdx.x - t.first[lo];
  const bool wide = kind & kWide;
  wait_for_predecessors();
  const Work a{t.e[lo], t.coef[lo], t.b1, t.c1, t.b2, t.c2, t.eps};
  switch (kind & (kParamMask | kGradFloat | kEight)) {
    case SO3LR_FLOAT32 | kGradFloat: return update_chunk<float, float, false>(a, chunk, wide);
    case SO3LR_FLOAT32 | kGradFloat | kEight: return update_chunk<float, float, true>(a, chunk, wide);
    case SO3LR_BFLOAT16: return update_chunk<__nv_bfloat16, __nv_bfloat16, false>(a, chunk, wide);
    case SO3LR_BFLOAT16 | kEight: return update_chunk<__nv_bfloat16, __nv_bfloat16, true>(a, chunk, wide);
    case SO3LR_BFLOAT16 | kGradFloat: return update_chunk<__nv_bfloat16, float, false>(a, chunk, wide);
    case SO3LR_BFLOAT16 | kGradFloat | kEight: return update_chunk<__nv_bfloat16, float, true>(a, chunk, wide);
    case SO3LR_FLOAT16: return update_chunk<__half, __half, false>(a, chunk, wide);
    case SO3LR_FLOAT16 | kEight: return update_chunk<__half, __half, true>(a, chunk, wide);
    case SO3LR_FLOAT16 | kGradFloat: return update_chunk<__half, float, false>(a, chunk, wide);
    case SO3LR_FLOAT16 | kGradFloat | kEight: return update_chunk<__half, float, true>(a, chunk, wide);
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
    const float top = a.scales[at / kScaleBlock];
    float f[kPer];
    if (wide && left == kPer) {
      values_of<SIGNED>(read_codes<true>(codes + at, left), top, f);
      write<true>(static_cast<O *>(a.values) + at, left, f);
    } else {
      values_of<SIGNED>(read_codes<false>(codes + at, left), top, f);
      write<false>(static_cast<O *>(a.values) + at, left, f);
    }
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
