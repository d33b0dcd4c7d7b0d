// AdamW over many tensors at once, moments in 32 bits or in 8.
//
//   m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr decay) - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)
//
// Bound by HBM: an element is read and written once (with a 16-bit parameter and a float32 master 28
// bytes with 32-bit moments, 16 with 8-bit ones). With 32-bit moments 268 M elements take 1090 us, 6.9
// TB/s; with 8-bit ones 317 M take 840 us, 6.0 TB/s, and under the power limit of a long run 957, 5.3.
// There neither fewer instructions (a third fewer: 850 -> 870 us), nor five blocks an SM (845, and the
// 32-bit step 1130), nor blocks of 2 or 4 times the elements (960 to 1300) help. Every tensor is cut into chunks of 2048
// elements, a chunk is a block's work, and one launch covers all tensors: a block finds
// its tensor in a table that travels as the kernel's argument, so that nothing is
// copied to the GPU before it and a captured graph holds its own table. The step
// counters live on the GPU: a first small kernel adds one to each and works out its
// bias corrections in float64, where 1 - beta^t keeps its digits for small t.
//
// An 8-bit moment is a code for each element and, for each 256 of them, the largest
// magnitude `top`: m = top t |t| with t = code / 127, v = top t^4 with t = code / 255.
// The roots spread the codes over the magnitudes that a block mixes: m down to 6e-5 of
// the largest, the root of v to 1.5e-5, both in steps of 1.6 % of the value near the
// largest, and the largest itself is kept exactly, so that a block decays as its
// moments do. Codes are rounded to nearest. A v that is not zero never becomes zero
// (its code is 1 at least): m / sqrt(v) would otherwise run away. One warp holds the 256
// elements of a scale, eight to a lane.
#include <algorithm>

#include "adamw.hpp"
#include "pairs.cuh"

namespace so3lr_b200 {
namespace {

constexpr int kChunk = 2048, kScaleBlock = 256, kPer = 8, kAdamThreads = kChunk / kPer;
constexpr int kAhead = 4 * kSmCount;  // chunks

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
  unsigned char kind[MOST];
  int count, chunks;
  const float4 *coef;   // of the first tensor, as the steps' kernel left it
  float b1, c1, b2, c2, eps;
};
// For each tensor lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), lr decay and, as an integer,
// its first chunk in its launch of k_adamw. Not 1 - lr decay: beside 1 one float32 would keep few
// of a small decay's digits (of 1e-7 it would make 1.19e-7, every step and element alike).
template <int MOST>
struct Steps {
  long long *step[MOST];
  int first[MOST];
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
                          float(lr * a.decay), __int_as_float(a.first[i]));
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

// What codes stand for. SIGNED: m, else v. Bytes become floats without the slow conversion: a
// byte in the low bits of 2^23.
template <bool SIGNED>
__device__ __forceinline__ void values_of(const Codes &codes, float top, float (&f)[kPer]) {
#pragma unroll
  for (int i = 0; i < kPer; i += 2) {
    const uint32_t word = SIGNED ? codes.word[i / 4] ^ 0x80808080u : codes.word[i / 4];
    const Pair code = Pair(__uint_as_float(__byte_perm(word, 0x4b000000u, 0x7440 + i % 4)),
                           __uint_as_float(__byte_perm(word, 0x4b000000u, 0x7441 + i % 4))) +
                      Pair(SIGNED ? -8388736.0f : -8388608.0f);
    const Pair t = code * Pair(SIGNED ? 1.0f / 127.0f : 1.0f / 255.0f), square = t * t;
    if (SIGNED) {
      float a, b;
      t.get(a, b);
      (square * Pair(top)).get(f[i], f[i + 1]);
      f[i] = copysignf(f[i], a);
      f[i + 1] = copysignf(f[i + 1], b);
    } else {
      (square * square * Pair(top)).get(f[i], f[i + 1]);
    }
  }
}
__device__ __forceinline__ float root(float v) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// The square roots of two numbers in 2^-126..1 as correctly rounded (but for one in a million,
// which is a unit off): Heron's step on x times the hardware's reciprocal root. With the
// approximate root alone one code in 30,000 would fall on the other side of a tie.
__device__ __forceinline__ Pair roots_of_shares(const Pair &x) {
  float a, b, ya, yb;
  x.get(a, b);
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(ya) : "f"(a));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(yb) : "f"(b));
  const Pair y(ya, yb), s = x * y;
  return madd(madd(s * Pair(-1.0f), s, x), y * Pair(0.5f), s);
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
__device__ __forceinline__ Pair shares_of(float a, float b, float inv) {
  float x, y;
  (Pair(a, b) * Pair(inv)).get(x, y);
  return Pair(fmaxf(fabsf(x), 0x1p-126f), fmaxf(fabsf(y), 0x1p-126f));
}
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
  // Pairs take an instruction for two elements (268 M elements in 8 bits 735 -> 692 us). Sums that
  // codes depend on are taken half by half: a contracted one is not the formula's in float32.
  auto sum = [](const Pair &x, const Pair &y, float &a, float &b) {
    float c, d;
    x.get(a, b);
    y.get(c, d);
    a = __fadd_rn(a, c);
    b = __fadd_rn(b, d);
  };
#pragma unroll
  for (int i = 0; i < kPer; i += 2) {
    const Pair gi(g[i], g[i + 1]);
    sum(Pair(a.b1) * Pair(m[i], m[i + 1]), Pair(a.c1) * gi, m[i], m[i + 1]);
    sum(Pair(a.b2) * Pair(v[i], v[i + 1]), Pair(a.c2) * (gi * gi), v[i], v[i + 1]);
  }
  // 1 - lr decay in two floats, so that p is rounded once. The second has the first's sign and is not 0,
  // so that an infinite p stays infinite: inf 0 and inf - inf would be NaN. (268 M elements in 8 bits 675
  // us with one float, 680 with two; 1092 with 32-bit moments in both forms.)
  const float keep = __fmul_rn(__fsub_rn(1.0f, coef.z), 1.0f - 0x1p-23f);
  const float keep_low = __fsub_rn(__fsub_rn(1.0f, keep), coef.z);
  // the denominators are at least eps, a normal number, and below 2^126
  auto move = [&](int i, const Pair &denominators) {
    float d, e;
    denominators.get(d, e);
    const Pair ratio = Pair(m[i], m[i + 1]) * Pair(reciprocal(d), reciprocal(e));
    const Pair old(p[i], p[i + 1]);
    madd(old, Pair(keep), madd(old, Pair(keep_low), ratio * Pair(-coef.x))).get(p[i], p[i + 1]);
  };
  auto move_by_root = [&] {
#pragma unroll
    for (int i = 0; i < kPer; i += 2) move(i, madd(Pair(root(v[i]), root(v[i + 1])), Pair(coef.y), Pair(a.eps)));
  };
  if (EIGHT) {
    bool m_live, v_live;
    const float m_top = scale_of(m, m_live), v_top = scale_of(v, v_live);
    float code[kPer];
    Codes cm{}, cv{};
    if (v_live) {  // the root of v is that of its share, which its code needs too
      const float inv = __frcp_rn(v_top), back = root(v_top) * coef.y;
#pragma unroll
      for (int i = 0; i < kPer; i += 2) {
        const Pair half = roots_of_shares(shares_of(v[i], v[i + 1], inv));
        move(i, madd(half, Pair(back), Pair(a.eps)));
        (roots_of_shares(half) * Pair(255.0f)).get(code[i], code[i + 1]);
        if (v[i] > 0.0f) code[i] = fmaxf(code[i], 1.0f);
        if (v[i + 1] > 0.0f) code[i + 1] = fmaxf(code[i + 1], 1.0f);
      }
      cv = pack(code);
    } else {
      move_by_root();
    }
    if (m_live) {
      const float inv = __frcp_rn(m_top);
#pragma unroll
      for (int i = 0; i < kPer; i += 2) {
        (roots_of_shares(shares_of(m[i], m[i + 1], inv)) * Pair(127.0f)).get(code[i], code[i + 1]);
        code[i] = copysignf(code[i], m[i]);
        code[i + 1] = copysignf(code[i + 1], m[i + 1]);
      }
      cm = pack(code);
    }
    write_codes<WHOLE>(static_cast<unsigned char *>(e.m) + at, left, cm);
    write_codes<WHOLE>(static_cast<unsigned char *>(e.v) + at, left, cv);
    if ((threadIdx.x & 31) == 0) {
      e.m_top[block] = m_top;
      e.v_top[block] = v_top;
    }
  } else {
    move_by_root();
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

// The tensor of a chunk, the last whose first chunk is not behind it: the warp's lanes look at
// every `every`-th, then at those up to the next.
template <int MOST>
__device__ __forceinline__ int tensor_of(const Table<MOST> &t, int chunk) {
  const int lane = threadIdx.x & 31, every = (t.count + 31) / 32;
  auto starts = [&](int i) { return i < t.count && __float_as_int(t.coef[i].w) <= chunk; };
  int lo = every * (31 - __clz(__ballot_sync(0xffffffffu, starts(lane * every))));
  if (MOST > 32 && every > 1) lo += 31 - __clz(__ballot_sync(0xffffffffu, lane < every && starts(lo + lane)));
  return lo;
}

template <int MOST>
__global__ void __launch_bounds__(kAdamThreads, 4) k_adamw(const __grid_constant__ Table<MOST> t) {
  dependents_may_start();
  wait_for_predecessors();
  const int block = int(blockIdx.x);
  const int lo = tensor_of(t, block);
  const float4 coef = t.coef[lo];
  const int kind = t.kind[lo];
  // The 8-bit step computes for longer than it loads: what a block of the next wave reads is on
  // its way to L2 meanwhile (67 M elements 219 us without, 190 with; the 32-bit step, bound by
  // HBM, has nothing of it: 268 M elements 1096 us without, 1110 with).
  if (threadIdx.x < 32 && block + kAhead < t.chunks) {
    const int then = tensor_of(t, block + kAhead), what = t.kind[then];
    const Entry &e = t.e[then];
    const long long at = (long long)(block + kAhead - __float_as_int(t.coef[then].w)) * kChunk;
    if ((what & kEight) && (what & kWide) && threadIdx.x < 4 && at + kChunk <= e.n) {
      const bool g = threadIdx.x == 0, p = threadIdx.x == 1;
      const void *from = g ? e.g : p ? (e.master ? e.master : e.p) : threadIdx.x == 2 ? e.m : e.v;
      const bool four = g ? what & kGradFloat : e.master || (what & kParamMask) == SO3LR_FLOAT32;
      const int size = g || p ? (four ? 4 : 2) : 1;
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(static_cast<const char *>(from) + at * size),
                   "r"(kChunk * size)
                   : "memory");
    }
  }
  const long long chunk = block - __float_as_int(coef.w);
  const bool wide = kind & kWide;
  const Work a{t.e[lo], coef, t.b1, t.c1, t.b2, t.c2, t.eps};
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

// values = what an 8-bit moment's codes stand for, 16 a thread
template <class O, bool SIGNED>
__global__ void __launch_bounds__(256) k_moment_values(const so3lr_moment_values_args a, bool wide) {
  dependents_may_start();
  const long long at = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 2 * kPer;
  if (at >= a.n) return;
  const unsigned char *codes = static_cast<const unsigned char *>(a.codes) + at;
  O *values = static_cast<O *>(a.values) + at;
  wait_for_predecessors();
  const float top = a.scales[at / kScaleBlock];
  float f[2][kPer];
  if (wide && at + 2 * kPer <= a.n) {
    const uint4 w = *reinterpret_cast<const uint4 *>(codes);
    values_of<SIGNED>(Codes{{w.x, w.y}}, top, f[0]);
    values_of<SIGNED>(Codes{{w.z, w.w}}, top, f[1]);
    write<true>(values, kPer, f[0]);
    write<true>(values + kPer, kPer, f[1]);
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int left = int(min((long long)kPer, a.n - at - h * kPer));  // may be negative
    values_of<SIGNED>(read_codes<false>(codes + h * kPer, left), top, f[h]);
    write<false>(values + h * kPer, left, f[h]);
  }
}

bool on(const void *p, std::size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <int MOST>
void launch_step(const so3lr_adamw_args &a, float4 *coef, cudaStream_t s) {
  static_assert(MOST <= 32 * 32, "a block's search takes two steps");
  Steps<MOST> steps{};
  steps.lr = a.lr;
  steps.lr_device = a.lr_device;
  steps.beta1 = a.beta1;
  steps.beta2 = a.beta2;
  steps.decay = a.weight_decay;
  Table<MOST> t{};
  t.b1 = float(a.beta1);
  t.c1 = float(1.0 - a.beta1);
  t.b2 = float(a.beta2);
  t.c2 = float(1.0 - a.beta2);
  t.eps = float(a.eps);
  auto flush = [&] {
    if (t.count) {
      t.coef = steps.coef = coef;
      steps.count = t.count;
      launch(k_adamw_steps<MOST>, unsigned((t.count + 31) / 32), 32, 0, s, steps);
      if (t.chunks) launch(k_adamw<MOST>, unsigned(t.chunks), kAdamThreads, 0, s, t);
    }
    coef += t.count;
    t.count = t.chunks = 0;
  };
  for (long long i = 0; i < a.count; ++i) {
    const so3lr_adamw_tensor &x = a.tensors[i];
    const long long chunks = (x.n + kChunk - 1) / kChunk;  // 2^29 at most
    if (t.count == MOST || t.chunks + chunks > 0x7fffffffLL - kAhead) flush();
    t.e[t.count] = Entry{x.param, x.grad, x.master, x.exp_avg, x.exp_avg_sq, x.exp_avg_scale, x.exp_avg_sq_scale, x.n};
    const bool wide = on(x.param, 16) && on(x.grad, 16) &&
                      on(x.master, 16) && on(x.exp_avg, 16) && on(x.exp_avg_sq, 16);
    t.kind[t.count] = static_cast<unsigned char>(x.dtype | (x.grad_dtype == SO3LR_FLOAT32 ? kGradFloat : 0) |
                                                 (x.exp_avg_scale ? kEight : 0) | (wide ? kWide : 0));
    steps.step[t.count] = x.step;
    steps.first[t.count] = t.chunks;
    t.chunks += int(chunks);
    ++t.count;
  }
  flush();
}

}  // namespace

long long adamw_bytes(const so3lr_adamw_args &a) { return a.count * (long long)sizeof(float4); }

// A table of 24 tensors (1.6 KB of arguments) where they fit: the driver copies the
// whole argument at every launch, 26 KB for 400 tensors.
void launch_adamw(const so3lr_adamw_args &a, void *workspace, cudaStream_t s) {
  float4 *coef = static_cast<float4 *>(workspace);
  if (a.count <= 24)
    launch_step<24>(a, coef, s);
  else
    launch_step<400>(a, coef, s);
}

void launch_moment_values(const so3lr_moment_values_args &a, cudaStream_t s) {
  const bool wide = on(a.codes, 16) && on(a.values, 16);
  const unsigned grid = unsigned((a.n + 512 * kPer - 1) / (512 * kPer));  // n <= 2^40: 2^28 blocks at most
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
