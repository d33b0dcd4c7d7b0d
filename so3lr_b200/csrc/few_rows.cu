// Dense products of the feed-forward layers for few rows (single atoms or tokens,
// small batches; the rule is in layers.hpp). All that counts is reading the weights
// once for each 16 rows, from HBM or, for small weights, from L2: a block takes 8
// output channels and its warps split the contraction, so that a 4096 x 4096 weight has
// 512 blocks; a long contraction to few channels is split over a cluster of blocks too.
// The products run on warp-level MMAs (m16n8k16 / m16n8k32, rows as M, channels as N)
// straight from registers: a tile of the tcgen05 kernel would be filled to a few of its
// 256 rows and would need its operands in shared memory first. One row through the
// 2048 x 8192 block takes 21 us, 4.7 TB/s of weights: two or three 16-byte loads a lane, held
// in registers, do not keep HBM busy.
//
// Contraction order: an MMA takes two 4-byte words of each lane's operands. A lane
// loads 16 contiguous bytes (words 0..3) of its row and of its channel at the same
// place, feeds words 0, 1 to one MMA and 2, 3 to the next; both operands use the
// same permutation of the contraction, so the sums are those of the formula.
#include "activation.cuh"
#include "block.hpp"
#include "layers_common.cuh"
#include "model_host.hpp"
#include "tensor_core.cuh"

namespace so3lr_b200 {
namespace {

__device__ __forceinline__ void mma_words(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_words(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_words(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1, signed char) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <class E, class Acc>
__device__ __forceinline__ void mma_step(Acc (&c)[4], const uint4 &x0, const uint4 &x1, const uint4 &w) {
  mma_words(c, x0.x, x1.x, x0.y, x1.y, w.x, w.y, E{});
  mma_words(c, x0.z, x1.z, x0.w, x1.w, w.z, w.w, E{});
}

// 16 bytes of a row from element k on. ALIGN: what rows start on (16 or 4 bytes, or 1).
// With 1 the 4-byte words around them are read and shifted, so the caller sees to it
// that the row has 4 bytes before and after.
template <class E, int ALIGN, bool WEIGHT>
__device__ __forceinline__ uint4 load_inside(const E *p, int k) {
  uint4 v;
  if (ALIGN == 16 && WEIGHT) {  // read once: not kept in L1. The kernel before may still be writing them: no .nc
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p + k)
                 : "memory");
  } else if (ALIGN == 16) {
    v = *reinterpret_cast<const uint4 *>(p + k);
  } else if (ALIGN == 4) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(p + k);
    v = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p + k), off = at % 4;
    const uint32_t *w = reinterpret_cast<const uint32_t *>(at - off);
    const uint32_t w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3], w4 = w[4], bits = 8 * uint32_t(off);
    v = make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits), __funnelshift_r(w2, w3, bits),
                   __funnelshift_r(w3, w4, bits));
  }
  return v;
}
// the same anywhere in the row, element by element; those past its end read as zero
template <class E>
__device__ __forceinline__ uint4 load_anywhere(const E *p, int k, int length) {
  constexpr int kPer = 16 / sizeof(E);
  alignas(16) E e[kPer] = {};
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (k + i < length) e[i] = p[k + i];
  return *reinterpret_cast<const uint4 *>(e);
}

constexpr int max_warps(bool two) { return two ? 8 : 16; }

struct FewArgs {
  int rows, n, k;
  const void *x;
  long long x_stride;
  const void *w, *w2;            // w2: the up projection (GATED)
  long long w_stride, w2_stride;
  void *y;
  long long y_stride;
  const float *a_scales, *b_scales, *bias;  // 8-bit products
  void *rest;                    // GATED: what y's rounding leaves of the hidden layer; LO: the same of x
  // LAYER
  const void *bias16, *residual; // a bias of the element type (`bias`: of float32)
  long long residual_stride;
  void *z;                       // optional: act's argument
  long long z_stride;
  int act;
};

// y = x w^T (8 bits: scaled), or silu(x w^T) * (x w2^T). TWO: more than 8 rows. LO: x is
// the sum of x and a.rest (rows like x's). The hidden layer is handed over in two
// 16-bit parts, so that its rounding does not show in y: with this few rows the second
// MMA costs nothing beside the weights' loads. LAYER: y = act(x w^T + bias) + residual.
template <class E, class O, bool GATED, bool LO, bool TWO, int ALIGN, bool LAYER>
__global__ void __launch_bounds__(32 * max_warps(TWO), TWO ? 3 : 2) k_few_rows(const FewArgs a) {
  constexpr bool kInt8 = std::is_same<E, signed char>::value;
  using Acc = typename std::conditional<kInt8, int, float>::type;
  constexpr int kPer = 16 / sizeof(E), kUnroll = ALIGN == 1 || GATED ? 2 : LO ? (TWO || ALIGN == 4 ? 2 : 3) : 4,
                kOut = GATED ? 2 : 1;
  __shared__ Acc part[max_warps(TWO)][kOut][TWO ? 16 : 8][8];
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // the blocks of a cluster share its channels and split the contraction
  const int splits = int(tc::cluster_size()), rank = int(tc::cluster_rank()), n0 = int(tc::cluster_index()) * 8;
  const int n = n0 + g, row0 = blockIdx.y * 16, rows = min(16, a.rows - row0);
  // lanes beyond the last row or channel read it again; their results are not written
  const int cn = min(n, a.n - 1);
  const E *w = static_cast<const E *>(a.w) + cn * a.w_stride, *w2 = static_cast<const E *>(a.w2) + cn * a.w2_stride;
  const E *x0 = static_cast<const E *>(a.x) + (row0 + min(g, rows - 1)) * a.x_stride;
  const E *x1 = static_cast<const E *>(a.x) + (row0 + min(g + 8, rows - 1)) * a.x_stride;
  const E *l0 = LO ? static_cast<const E *>(a.rest) + (x0 - static_cast<const E *>(a.x)) : nullptr;
  const E *l1 = LO ? static_cast<const E *>(a.rest) + (x1 - static_cast<const E *>(a.x)) : nullptr;
  const int steps = (a.k + 4 * kPer - 1) / (4 * kPer);
  const int which = rank * warps + warp, all = splits * warps;
  const int begin = int((long long)steps * which / all), end = int((long long)steps * (which + 1) / all);
  dependents_may_start();
  // the first weights on their way to L2, which needs no order with the kernel before
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int k = ((begin + i) * 4 + t) * kPer;
    if (begin + i < end && k < a.k) {
      asm volatile("prefetch.global.L2 [%0];" ::"l"(w + k));
      if (GATED) asm volatile("prefetch.global.L2 [%0];" ::"l"(w2 + k));
    }
  }
  wait_for_predecessors();
  Acc acc[kOut][4] = {};
  const uint4 zero = make_uint4(0, 0, 0, 0);
  auto multiply = [&](const uint4 &v0, const uint4 &v1, const uint4 &r0, const uint4 &r1, const uint4 &vw,
                      const uint4 &vw2) {
    mma_step<E>(acc[0], v0, TWO ? v1 : zero, vw);
    if (LO) mma_step<E>(acc[0], r0, TWO ? r1 : zero, vw);
    if (GATED) mma_step<E>(acc[kOut - 1], v0, TWO ? v1 : zero, vw2);
  };
  auto step_anywhere = [&](int st) {
    const int k = (st * 4 + t) * kPer;
    uint4 vw = zero, vw2 = zero, v0 = zero, v1 = zero, r0 = zero, r1 = zero;
    if (k < a.k) {
      vw = load_anywhere(w, k, a.k);
      if (GATED) vw2 = load_anywhere(w2, k, a.k);
      v0 = load_anywhere(x0, k, a.k);
      if (TWO) v1 = load_anywhere(x1, k, a.k);
      if (LO) r0 = load_anywhere(l0, k, a.k);
      if (LO && TWO) r1 = load_anywhere(l1, k, a.k);
    }
    multiply(v0, v1, r0, r1, vw, vw2);
  };
  auto steps_inside = [&](int st, auto count) {  // `count` steps, all four lanes of a row inside it
    constexpr int C = decltype(count)::value;
    const int k = (st * 4 + t) * kPer;
    uint4 vw[C], vw2[GATED ? C : 1], v0[C], v1[TWO ? C : 1], r0[LO ? C : 1], r1[LO && TWO ? C : 1];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      vw[i] = load_inside<E, ALIGN, true>(w, k + i * 4 * kPer);
      if (GATED) vw2[i] = load_inside<E, ALIGN, true>(w2, k + i * 4 * kPer);
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      v0[i] = load_inside<E, ALIGN, false>(x0, k + i * 4 * kPer);
      if (TWO) v1[i] = load_inside<E, ALIGN, false>(x1, k + i * 4 * kPer);
      if (LO) r0[i] = load_inside<E, ALIGN, false>(l0, k + i * 4 * kPer);
      if (LO && TWO) r1[i] = load_inside<E, ALIGN, false>(l1, k + i * 4 * kPer);
    }
#pragma unroll
    for (int i = 0; i < C; ++i)
      multiply(v0[i], TWO ? v1[i] : zero, LO ? r0[i] : zero, LO && TWO ? r1[i] : zero, vw[i], GATED ? vw2[i] : zero);
  };
  // loads of 16 bytes where they are inside the row (and, off the boundaries, 4 bytes before and after them)
  constexpr int kAround = ALIGN == 1 ? 4 / int(sizeof(E)) : 0;
  int st = begin;
  if (ALIGN == 1 && st == 0 && st < end) step_anywhere(st++);
  const int whole = min(end, (a.k - kAround) / (4 * kPer));
  for (; st + kUnroll <= whole; st += kUnroll) steps_inside(st, std::integral_constant<int, kUnroll>{});
  for (; st < whole; ++st) steps_inside(st, std::integral_constant<int, 1>{});
  for (; st < end; ++st) step_anywhere(st);
#pragma unroll
  for (int o = 0; o < kOut; ++o) {
    part[warp][o][g][2 * t] = acc[o][0];
    part[warp][o][g][2 * t + 1] = acc[o][1];
    if (TWO) {
      part[warp][o][g + 8][2 * t] = acc[o][2];
      part[warp][o][g + 8][2 * t + 1] = acc[o][3];
    }
  }
  __syncthreads();
  int parts = warps;
  if (splits > 1) {  // all into the first part of the first block
    parts = 1;
    const int i = threadIdx.x, row = i >> 3, c = i & 7;  // 8 warps or more: a thread has one sum at most
    if (i < 8 * rows)
#pragma unroll
      for (int o = 0; o < kOut; ++o) {
        Acc sum{};
        for (int k = 0; k < warps; ++k) sum += part[k][o][row][c];
        part[0][o][row][c] = sum;
      }
    __syncwarp();
    tc::cluster_sync();
    if (rank == 0 && i < 8 * rows)
#pragma unroll
      for (int o = 0; o < kOut; ++o) {
        Acc sum = part[0][o][row][c];
        for (int k = 1; k < splits; ++k) sum += tc::load_of_rank(&part[0][o][row][c], k);
        part[0][o][row][c] = sum;
      }
    __syncwarp();
    tc::cluster_sync();  // no block leaves before its sums are read
    if (rank != 0) return;
  }
  for (int i = threadIdx.x; i < 8 * rows; i += blockDim.x) {
    const int row = i >> 3, c = n0 + (i & 7);
    if (c >= a.n) continue;
    Acc sum[kOut] = {};
    for (int k = 0; k < parts; ++k)
#pragma unroll
      for (int o = 0; o < kOut; ++o) sum[o] += part[k][o][row][i & 7];
    float y;
    if (kInt8)
      y = fmaf(float(sum[0]) * a.a_scales[row0 + row], a.b_scales[c], a.bias ? a.bias[c] : 0.0f);
    else if (GATED)
      y = silu_f32(float(sum[0])) * float(sum[kOut - 1]);
    else
      y = float(sum[0]);
    if constexpr (LAYER) {
      y += a.bias ? a.bias[c] : a.bias16 ? to_float(static_cast<const O *>(a.bias16)[c]) : 0.0f;
      if (a.z) static_cast<O *>(a.z)[(row0 + row) * a.z_stride + c] = kept<O>(y);
      by_activation(a.act, [&](auto act) { y = activate<decltype(act)::value>(y); });
      if (a.residual) y += to_float(static_cast<const O *>(a.residual)[(row0 + row) * a.residual_stride + c]);
    }
    const O rounded = from_float<O>(y);
    static_cast<O *>(a.y)[(row0 + row) * a.y_stride + c] = rounded;
    if (GATED) {  // nothing is left of an infinity or a NaN
      const float rest = y - to_float(rounded);
      static_cast<O *>(a.rest)[(long long)(row0 + row) * a.y_stride + c] =
          from_float<O>(fabsf(rest) < 1e30f ? rest : 0.0f);
    }
  }
}

bool rows_on(int bytes, const void *p, long long stride, long long rows, int size) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && (rows == 1 || stride * size % bytes == 0));
}

template <class E, class O, bool GATED, bool LO, bool LAYER = false>
void run(const FewArgs &a, cudaStream_t s) {
  constexpr int kPer = 16 / sizeof(E);
  auto all_on = [&](int bytes) {
    constexpr int e = sizeof(E);
    return rows_on(bytes, a.x, a.x_stride, a.rows, e) && rows_on(bytes, a.w, a.w_stride, a.n, e) &&
           rows_on(bytes, a.w2, a.w2_stride, a.n, e) && (!LO || rows_on(bytes, a.rest, a.x_stride, a.rows, e));
  };
  // Warps that split the contraction, four steps of 64 bytes or more to each: 8, or 16
  // where the blocks alone would leave too few loads in flight. One row, 2048 channels
  // of 8192 bfloat16 (256 blocks): 12.3 us with 8, 9.3 us with 16; 4096 channels of
  // 4096 bytes (512 blocks): 4.4 us with 8, 6.5 us with 16.
  const unsigned channels = unsigned((a.n + 7) / 8), groups = unsigned((a.rows + 15) / 16), blocks = channels * groups;
  const int most = blocks < 2 * kSmCount ? max_warps(a.rows > 8) : 8;
  const int steps = (a.k + 4 * kPer - 1) / (4 * kPer), warps = std::max(1, std::min(most, steps / 4));
  // Up to 8 blocks in a cluster split it too where SMs would be idle and each warp would have 12 steps or
  // more (16 rows through the 64 x 8192 block: 16.7 us without, 7.6 with; where a warp has 8, 256 channels
  // of 4096 bytes, a cluster costs what it gives: 3.0 and 3.2 us).
  unsigned splits = 1;
  while (splits < 8 && blocks * splits < kSmCount && steps >= 12 * int(splits) * warps) splits *= 2;
  auto go = [&](auto align) {
    constexpr int A = decltype(align)::value;
    launch_clusters(a.rows > 8 ? &k_few_rows<E, O, GATED, LO, true, A, LAYER> : &k_few_rows<E, O, GATED, LO, false, A, LAYER>,
                    dim3(channels * splits, groups), unsigned(32 * warps), splits > 1 ? splits : 0, 0, s, a);
  };
  if (all_on(16))
    go(std::integral_constant<int, 16>{});
  else if (all_on(4))
    go(std::integral_constant<int, 4>{});
  else
    go(std::integral_constant<int, 1>{});
}

}  // namespace

void launch_int8_linear_few(const so3lr_int8_linear_args &l, cudaStream_t s) {
  const FewArgs a{int(l.rows), int(l.n), int(l.k), l.a, l.a_stride, l.b, nullptr, l.b_stride, 0, l.y, l.y_stride,
                  l.a_scales, l.b_scales, l.bias, nullptr};
  if (l.out_dtype == SO3LR_FLOAT32)
    run<signed char, float, false, false>(a, s);
  else if (l.out_dtype == SO3LR_BFLOAT16)
    run<signed char, __nv_bfloat16, false, false>(a, s);
  else
    run<signed char, __half, false, false>(a, s);
}

void launch_feed_forward_few(const so3lr_feed_forward_args &f, void *h, long long h_stride, void *h_rest,
                             cudaStream_t s) {
  const FewArgs up{int(f.rows), int(f.hidden), int(f.width), f.x, f.x_stride, f.w_gate, f.w_up, f.w_gate_stride,
                   f.w_up_stride, h, h_stride, nullptr, nullptr, nullptr, h_rest};
  const FewArgs down{int(f.rows), int(f.width), int(f.hidden), h, h_stride, f.w_down, nullptr, f.w_down_stride, 0,
                     f.y, f.y_stride, nullptr, nullptr, nullptr, h_rest};
  if (f.dtype == SO3LR_BFLOAT16) {
    run<__nv_bfloat16, __nv_bfloat16, true, false>(up, s);
    run<__nv_bfloat16, __nv_bfloat16, false, true>(down, s);
  } else {
    run<__half, __half, true, false>(up, s);
    run<__half, __half, false, true>(down, s);
  }
}

void launch_linear_few(const so3lr_linear_args &l, cudaStream_t s) {
  FewArgs a{int(l.rows), int(l.n), int(l.k), l.x, l.x_stride, l.w, nullptr, l.w_stride, 0, l.y, l.y_stride};
  if (l.bias_dtype == SO3LR_FLOAT32)
    a.bias = static_cast<const float *>(l.bias);
  else
    a.bias16 = l.bias;
  a.residual = l.residual;
  a.residual_stride = l.residual_stride;
  a.z = l.z;
  a.z_stride = l.z_stride;
  a.act = l.activation;
  if (l.dtype == SO3LR_BFLOAT16)
    run<__nv_bfloat16, __nv_bfloat16, false, false, true>(a, s);
  else
    run<__half, __half, false, false, true>(a, s);
}

}  // namespace so3lr_b200
