// Elementwise part of the dense layer's gradient: dz = dy act'(z) in the element type, as the
// products after it read it, and the bias gradient, its column sums in float32 before that
// rounding.
//
// Bound by HBM (dy and z in, dz out): 8192 x 8192 bfloat16 70 us, 5.8 TB/s; rows off the boundaries, dy
// one element at a time, 3.4 to 4.2 TB/s. With an activation what is read here is not read again and is not
// kept in L2 for it: dz is, and the two products that follow find it there (a whole step of 24000 x 256 -> 1024
// 114 us without, 107 with). Without one dy is dz, and only its column sums are formed here: its loads are
// ordinary (24000 x 256 -> 1024 with a bias, backward, 62 us marked as first to be evicted, 61 so; 8192 x 4096 ->
// 4096 after a kernel that wrote dy 392 and 381). A warp takes 256 columns of a row, or several rows of
// narrow ones, 8 columns a lane; a block walks down its share of the rows and writes one row
// of sums, which k_bias_sum adds in order.
#include <algorithm>

#include "activation.cuh"
#include "block.hpp"

namespace so3lr_b200 {
namespace {

constexpr int kVec = 8, kWarps = 8;

struct BackArgs {
  long long rows, rows_per_block;
  int n, lanes;               // lanes: of a warp that share a row, a power of two
  const void *dy, *z;
  long long dy_stride, z_stride;
  void *dz;                   // nullptr: dy itself is dz
  long long dz_stride;
  float *partial;             // [blocks of a column strip][n], or nullptr
  bool dy_wide, z_wide;       // rows on 16-byte boundaries
};

// ONCE: no kernel after this one reads it
template <bool WIDE, bool ONCE, class T>
__device__ __forceinline__ Chunk<T, kVec> load_part(const T *p, bool wide, int left) {
  if (WIDE && ONCE) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(p));
    return *reinterpret_cast<const Chunk<T, kVec> *>(&v);
  }
  if (WIDE || (wide && left >= kVec)) return load_chunk<T, kVec>(p);
  Chunk<T, kVec> c;
#pragma unroll
  for (int i = 0; i < kVec; ++i) c.e[i] = i < left ? p[i] : from_float<T>(0.0f);
  return c;
}

// WIDE: all rows on 16-byte boundaries and of whole chunks
template <class T, int ACT, bool WIDE>
__global__ void __launch_bounds__(32 * kWarps) k_linear_backward(const BackArgs a) {
  constexpr bool kOnce = ACT != SO3LR_NO_ACTIVATION;  // else there is no z, and dy is dz, which the products read next
  __shared__ float sums[kWarps * 32][kVec + 1];
  dependents_may_start();
  wait_for_predecessors();
  const int lane = threadIdx.x & 31, t = lane % a.lanes, rows_of_warp = 32 / a.lanes;
  const int c = (blockIdx.x * a.lanes + t) * kVec, left = a.n - c;
  const int step = kWarps * rows_of_warp;
  const long long begin = blockIdx.y * a.rows_per_block, end = min(a.rows, begin + a.rows_per_block);
  Floats<kVec> sum;
#pragma unroll
  for (int i = 0; i < kVec / 2; ++i) sum.v[i] = Pair(0.0f);
  auto one = [&](const Chunk<T, kVec> &dy, const Chunk<T, kVec> &z, long long row) {
    Floats<kVec> d = floats_of(dy);
    const Floats<kVec> zf = floats_of(z);
#pragma unroll
    for (int i = 0; i < kVec / 2; ++i) {
      if (ACT != SO3LR_NO_ACTIVATION) d.v[i] = d.v[i] * slope<ACT>(zf.v[i]);
      sum.v[i] = sum.v[i] + d.v[i];
    }
    if (ACT == SO3LR_NO_ACTIVATION) return;
    T *dz = static_cast<T *>(a.dz) + row * a.dz_stride + c;  // rows are padded to whole chunks
    store_chunk<T, kVec>(dz, chunk_of_floats<T, kVec>(d));
  };
  if (left > 0) {
    const T *dy = static_cast<const T *>(a.dy) + c, *z = static_cast<const T *>(a.z) + c;
    long long row = begin + (threadIdx.x >> 5) * rows_of_warp + lane / a.lanes;
    constexpr int kAtOnce = WIDE ? 4 : 1;
    for (; row + (kAtOnce - 1) * step < end; row += kAtOnce * step) {
      Chunk<T, kVec> cd[kAtOnce], cz[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        cd[k] = load_part<WIDE, kOnce>(dy + (row + k * step) * a.dy_stride, a.dy_wide, left);
        if (kOnce) cz[k] = load_part<WIDE, kOnce>(z + (row + k * step) * a.z_stride, a.z_wide, left);
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) one(cd[k], cz[k], row + k * step);
    }
    for (; row < end; row += step) {
      const Chunk<T, kVec> cd = load_part<WIDE, kOnce>(dy + row * a.dy_stride, a.dy_wide, left);
      Chunk<T, kVec> cz{};
      if (kOnce) cz = load_part<WIDE, kOnce>(z + row * a.z_stride, a.z_wide, left);
      one(cd, cz, row);
    }
  }
  if (!a.partial) return;
  const Chunk<float, kVec> total = chunk_of_floats<float, kVec>(sum);
#pragma unroll
  for (int i = 0; i < kVec; ++i) sums[threadIdx.x][i] = total.e[i];
  __syncthreads();
  // thread: one column of the strip; the rows' owners in order
  for (int i = threadIdx.x; i < a.lanes * kVec; i += blockDim.x) {
    const int column = blockIdx.x * a.lanes * kVec + i;
    if (column >= a.n) break;
    float all = 0.0f;
    for (int k = i / kVec; k < kWarps * 32; k += a.lanes) all += sums[k][i % kVec];
    a.partial[(size_t)blockIdx.y * a.n + column] = all;
  }
}

template <class B>
__global__ void k_bias_sum(int parts, int n, const float *partial, B *out) {
  __shared__ float part[32][33];
  dependents_may_start();
  wait_for_predecessors();
  const int c = blockIdx.x * 32 + threadIdx.x;
  float total = 0.0f;
  if (c < n)
#pragma unroll 8
    for (int k = threadIdx.y; k < parts; k += 32) total += partial[(size_t)k * n + c];
  part[threadIdx.y][threadIdx.x] = total;
  __syncthreads();
  if (threadIdx.y == 0 && c < n) {
    total = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; ++k) total += part[k][threadIdx.x];
    out[c] = from_float<B>(total);
  }
}

struct Plan {
  int lanes, strips, parts;
  long long rows_per_block;
};
Plan plan(long long rows, long long n) {
  Plan p;
  p.lanes = 1;
  while (p.lanes < 32 && p.lanes * kVec < n) p.lanes *= 2;
  p.strips = int((n + p.lanes * kVec - 1) / (p.lanes * kVec));
  // about eight blocks an SM in all, a row for each warp at least
  const long long least = (long long)kWarps * (32 / p.lanes);
  const long long want = std::max<long long>(1, 8LL * kSmCount / p.strips);
  p.rows_per_block = std::max(least, (rows + want - 1) / want);
  p.parts = int((rows + p.rows_per_block - 1) / p.rows_per_block);
  return p;
}
bool wide(const void *p, long long stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0; }

}  // namespace

long long linear_elementwise_bytes(const so3lr_linear_backward_args &a) {
  return a.dbias && a.rows > 0 ? (long long)plan(a.rows, a.n).parts * a.n * 4 : 0;
}

void launch_linear_elementwise(const so3lr_linear_backward_args &a, void *dz, long long dz_stride, float *partial,
                               cudaStream_t s) {
  const Plan p = plan(a.rows, a.n);
  const BackArgs b{a.rows, p.rows_per_block, int(a.n), p.lanes, a.dy, a.z, a.dy_stride, a.z_stride, dz, dz_stride,
                   partial, wide(a.dy, a.dy_stride), wide(a.z, a.z_stride)};
  auto go = [&](auto t) {
    using T = decltype(t);
    auto by_width = [&](auto act) {
      constexpr int A = decltype(act)::value;
      return b.dy_wide && (A == SO3LR_NO_ACTIVATION || b.z_wide) && a.n % kVec == 0 ? &k_linear_backward<T, A, true>
                                                                                   : &k_linear_backward<T, A, false>;
    };
    using std::integral_constant;
    void (*kernel)(BackArgs) = a.activation == SO3LR_SILU        ? by_width(integral_constant<int, SO3LR_SILU>{})
                               : a.activation == SO3LR_GELU      ? by_width(integral_constant<int, SO3LR_GELU>{})
                               : a.activation == SO3LR_GELU_TANH ? by_width(integral_constant<int, SO3LR_GELU_TANH>{})
                               : a.activation == SO3LR_RELU      ? by_width(integral_constant<int, SO3LR_RELU>{})
                                                                 : by_width(integral_constant<int, SO3LR_NO_ACTIVATION>{});
    launch(kernel, dim3(p.strips, p.parts), 32 * kWarps, 0, s, b);
    if (!partial) return;
    const dim3 grid(unsigned((a.n + 31) / 32)), block(32, 32);
    if (a.bias_dtype == SO3LR_FLOAT32)
      launch(k_bias_sum<float>, grid, block, 0, s, p.parts, int(a.n), partial, static_cast<float *>(a.dbias));
    else
      launch(k_bias_sum<T>, grid, block, 0, s, p.parts, int(a.n), partial, static_cast<T *>(a.dbias));
  };
  if (a.dtype == SO3LR_BFLOAT16)
    go(__nv_bfloat16{});
  else
    go(__half{});
}

}  // namespace so3lr_b200
