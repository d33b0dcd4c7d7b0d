// Row kernels of the feed-forward layers: RMS norm with the residual's addition
// (forward, 8-bit output, backward), the 8-bit gate and the reading back of 8-bit
// rows. All are bound by HBM: every input element is read once into registers,
// every output written once; the row statistics are reduced between the two.
//
// A row belongs to one warp (up to 16 elements per lane, so that short rows need
// no block barrier) or to one block. A thread holds N chunks of VEC elements:
// 16-byte chunks where every row starts on a 16-byte boundary, single elements
// otherwise (odd widths, views).
#include "layers_common.cuh"
#include "model_host.hpp"

namespace so3lr_b200 {
namespace {

constexpr int kWarpRows = 8;     // rows of a block when a warp owns a row
constexpr int kPerThread = 16;   // elements a thread holds at most (norm)

// The threads of one row: a warp or the whole block. Reductions run in a fixed
// order and return the same value to every thread of the row.
template <bool WARP>
struct RowTeam {
  int t, size;
  __device__ RowTeam() : t(WARP ? threadIdx.x & 31 : threadIdx.x), size(WARP ? 32 : blockDim.x) {}
  // slot: 32 floats of shared memory that no other pending reduction uses
  __device__ __forceinline__ float sum(float v, float *slot) const {
    v = warp_sum(v);
    if (WARP) return v;
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    float total = 0.0f;
    for (int i = 0; i < warps; ++i) total += slot[i];
    return total;
  }
  __device__ __forceinline__ float2 sum2(float a, float b, float2 *slot) const {
    a = warp_sum(a);
    b = warp_sum(b);
    if (WARP) return make_float2(a, b);
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    float2 total = make_float2(0.0f, 0.0f);
    for (int i = 0; i < warps; ++i) {
      total.x += slot[i].x;
      total.y += slot[i].y;
    }
    return total;
  }
  __device__ __forceinline__ uint32_t max(uint32_t v, uint32_t *slot) const {
    v = __reduce_max_sync(0xffffffffu, v);
    if (WARP) return v;
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    uint32_t top = 0;
    for (int i = 0; i < warps; ++i) top = ::max(top, slot[i]);
    return top;
  }
};

// y = s w rstd, s = x + residual as stored. QUANT: y goes to 8 bits with the row's scale.
template <class T, class W, int VEC, int N, bool WARP, bool QUANT>
__global__ void __launch_bounds__(WARP ? 32 * kWarpRows : 1024) k_rms_norm(const so3lr_rms_norm_args a) {
  __shared__ float slot[32];
  __shared__ uint32_t slot_max[32];
  const RowTeam<WARP> team;
  const long long row = WARP ? (long long)blockIdx.x * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.rows) return;  // whole warps (WARP) only: a block row always exists
  const int width = int(a.width);
  const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
  const T *r = a.residual ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
  const W *w = static_cast<const W *>(a.weight);

  Chunk<T, VEC> cx[N], cr[N];
  Chunk<W, VEC> cw[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * team.size + team.t) * VEC;
    if (c < width) {
      cx[j] = load_chunk<T, VEC>(x + c);
      if (r) cr[j] = load_chunk<T, VEC>(r + c);
      cw[j] = load_chunk<W, VEC>(w + c);
    }
  }
  float v[N * VEC], sq = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * team.size + team.t) * VEC;
    if (c < width) {
      if (r) {
        // the stream is kept in the element type, and the norm is of what is kept
#pragma unroll
        for (int i = 0; i < VEC; ++i) cx[j].e[i] = from_float<T>(to_float(cx[j].e[i]) + to_float(cr[j].e[i]));
        store_chunk<T, VEC>(static_cast<T *>(a.s) + row * a.s_stride + c, cx[j]);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[j * VEC + i] = to_float(cx[j].e[i]);
        sq = fmaf(v[j * VEC + i], v[j * VEC + i], sq);
      }
    }
  }
  const float rstd = 1.0f / sqrtf(team.sum(sq, slot) / float(width) + float(a.eps));
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * team.size + team.t) * VEC;
    if (c < width) {
      Chunk<T, VEC> out;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float y = v[j * VEC + i] * rstd * to_float(cw[j].e[i]);
        v[j * VEC + i] = y;
        if (QUANT)
          top = ::max(top, __float_as_uint(y) & 0x7fffffffu);
        else
          out.e[i] = from_float<T>(y);
      }
      if (!QUANT) store_chunk<T, VEC>(static_cast<T *>(a.y) + row * a.y_stride + c, out);
    }
  }
  if (!QUANT) return;
  float inv;
  const float scale = row_scale(team.max(top, slot_max), inv);
  if (team.t == 0) a.scales[row] = scale;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * team.size + team.t) * VEC;
    if (c < width) {
      Chunk<signed char, VEC> out;
#pragma unroll
      for (int i = 0; i < VEC; ++i) out.e[i] = to_code(v[j * VEC + i], inv);
      store_chunk<signed char, VEC>(a.codes + row * a.codes_stride + c, out);
    }
  }
}

// dx = rstd (a - xh mean(a xh)) + ds with a = dy w, xh = s rstd; each block also
// sums dy xh over its rows (a fixed set, in order) into one row of `partial`.
template <class T, class W, int VEC, int N, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kWarpRows : 1024) k_rms_norm_backward(const so3lr_rms_norm_backward_args a, float *__restrict__ partial) {
  __shared__ float2 slot[2][32];
  extern __shared__ float column[];  // WARP: kWarpRows x width
  const RowTeam<WARP> team;
  const int width = int(a.width);
  const int teams = WARP ? kWarpRows : 1, team_id = WARP ? threadIdx.x >> 5 : 0;
  Chunk<W, VEC> cw[N];
  float dw[N * VEC];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * team.size + team.t) * VEC;
    if (c < width) cw[j] = load_chunk<W, VEC>(static_cast<const W *>(a.weight) + c);
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[j * VEC + i] = 0.0f;
  }
  int parity = 0;
  for (long long row = (long long)blockIdx.x * teams + team_id; row < a.rows; row += (long long)gridDim.x * teams) {
    const T *s = static_cast<const T *>(a.s) + row * a.s_stride;
    const T *dy = static_cast<const T *>(a.dy) + row * a.dy_stride;
    const T *ds = a.ds ? static_cast<const T *>(a.ds) + row * a.ds_stride : nullptr;
    Chunk<T, VEC> cs[N], cd[N], ce[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * team.size + team.t) * VEC;
      if (c < width) {
        cs[j] = load_chunk<T, VEC>(s + c);
        cd[j] = load_chunk<T, VEC>(dy + c);
        if (ds) ce[j] = load_chunk<T, VEC>(ds + c);
      }
    }
    float sq = 0.0f, dot = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * team.size + team.t) * VEC;
      if (c < width) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float f = to_float(cs[j].e[i]);
          sq = fmaf(f, f, sq);
          dot = fmaf(f, to_float(cd[j].e[i]) * to_float(cw[j].e[i]), dot);
        }
      }
    }
    const float2 total = team.sum2(sq, dot, slot[parity]);
    parity ^= 1;
    const float rstd = 1.0f / sqrtf(total.x / float(width) + float(a.eps));
    const float mean = total.y * rstd / float(width);  // mean(a xh)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * team.size + team.t) * VEC;
      if (c < width) {
        Chunk<T, VEC> out;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float xh = to_float(cs[j].e[i]) * rstd, d = to_float(cd[j].e[i]);
          dw[j * VEC + i] = fmaf(d, xh, dw[j * VEC + i]);
          float g = rstd * (d * to_float(cw[j].e[i]) - xh * mean);
          if (ds) g += to_float(ce[j].e[i]);
          out.e[i] = from_float<T>(g);
        }
        store_chunk<T, VEC>(static_cast<T *>(a.dx) + row * a.dx_stride + c, out);
      }
    }
  }
  if (!WARP) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * team.size + team.t) * VEC;
      if (c < width)
#pragma unroll
        for (int i = 0; i < VEC; ++i) partial[(size_t)blockIdx.x * width + c + i] = dw[j * VEC + i];
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * team.size + team.t) * VEC;
    if (c < width)
#pragma unroll
      for (int i = 0; i < VEC; ++i) column[team_id * width + c + i] = dw[j * VEC + i];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < width; c += blockDim.x) {
    float total = 0.0f;
#pragma unroll
    for (int k = 0; k < kWarpRows; ++k) total += column[k * width + c];
    partial[(size_t)blockIdx.x * width + c] = total;
  }
}

// column sums of `partial` (nparts x width) in a fixed order: 32 columns per
// block, part k summed by thread row k % 32, then the 32 thread rows in order
template <class W>
__global__ void k_column_sum(int nparts, int width, const float *__restrict__ partial, W *__restrict__ out) {
  __shared__ float part[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float total = 0.0f;
  if (c < width)
#pragma unroll 4
    for (int k = threadIdx.y; k < nparts; k += 32) total += partial[(size_t)k * width + c];
  part[threadIdx.y][threadIdx.x] = total;
  __syncthreads();
  if (threadIdx.y == 0 && c < width) {
    total = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; ++k) total += part[k][threadIdx.x];
    out[c] = from_float<W>(total);
  }
}

template <class T, int VEC, int N, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kWarpRows : 1024) k_gate_int8(const so3lr_gate_int8_args a) {
  __shared__ uint32_t slot[32];
  const RowTeam<WARP> team;
  const long long row = WARP ? (long long)blockIdx.x * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.rows) return;
  const int hidden = int(a.hidden);
  const T *g = static_cast<const T *>(a.gu) + row * a.gu_stride, *u = g + hidden;
  Chunk<T, VEC> cg[N], cu[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * team.size + team.t) * VEC;
    if (c < hidden) {
      cg[j] = load_chunk<T, VEC>(g + c);
      cu[j] = load_chunk<T, VEC>(u + c);
    }
  }
  float v[N * VEC];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * team.size + team.t) * VEC;
    if (c < hidden) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[j * VEC + i] = silu_f32(to_float(cg[j].e[i])) * to_float(cu[j].e[i]);
        top = ::max(top, __float_as_uint(v[j * VEC + i]) & 0x7fffffffu);
      }
    }
  }
  float inv;
  const float scale = row_scale(team.max(top, slot), inv);
  if (team.t == 0) a.scales[row] = scale;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * team.size + team.t) * VEC;
    if (c < hidden) {
      Chunk<signed char, VEC> out;
#pragma unroll
      for (int i = 0; i < VEC; ++i) out.e[i] = to_code(v[j * VEC + i], inv);
      store_chunk<signed char, VEC>(a.codes + row * a.codes_stride + c, out);
    }
  }
}

template <class T, int VEC>
__global__ void k_dequantize_int8(const so3lr_dequantize_int8_args a) {
  const long long per_row = a.width / VEC, total = a.rows * per_row;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const long long row = total < (1LL << 31) ? uint32_t(i) / uint32_t(per_row) : i / per_row;
    const long long c = (i - row * per_row) * VEC;
    const float scale = a.scales[row];
    const Chunk<signed char, VEC> q = load_chunk<signed char, VEC>(a.codes + row * a.codes_stride + c);
    Chunk<T, VEC> out;
#pragma unroll
    for (int k = 0; k < VEC; ++k) out.e[k] = from_float<T>(float(q.e[k]) * scale);
    store_chunk<T, VEC>(static_cast<T *>(a.out) + row * a.out_stride + c, out);
  }
}

// ------------------------------------------------------------------ dispatch
bool aligned(const void *p, long long stride, int size, int bytes) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && (stride * size) % bytes == 0);
}

// Threads that hold a row of `width` elements, PER of them each: a warp where one
// suffices, else a block of whole warps.
int row_threads(long long width, int per) { return int((width + 32LL * per - 1) / (32LL * per)) * 32; }

template <class F>
void by_type(int dtype, F &&f) {
  if (dtype == SO3LR_FLOAT32)
    f(float{});
  else if (dtype == SO3LR_BFLOAT16)
    f(__nv_bfloat16{});
  else
    f(__half{});
}
template <class T, class F>
void by_weight(int dtype, int weight_dtype, F &&f) {
  if (weight_dtype == SO3LR_FLOAT32 && dtype != SO3LR_FLOAT32)
    f(float{});
  else
    f(T{});
}

template <class T, class W, int VEC, int N>
void norm_forward(const so3lr_rms_norm_args &a, cudaStream_t s) {
  const int threads = row_threads(a.width, VEC * N);
  const bool warp = threads == 32;
  const unsigned grid = unsigned(warp ? (a.rows + kWarpRows - 1) / kWarpRows : a.rows);
  const int block = warp ? 32 * kWarpRows : threads;
  if (warp && a.codes)
    k_rms_norm<T, W, VEC, N, true, true><<<grid, block, 0, s>>>(a);
  else if (warp)
    k_rms_norm<T, W, VEC, N, true, false><<<grid, block, 0, s>>>(a);
  else if (a.codes)
    k_rms_norm<T, W, VEC, N, false, true><<<grid, block, 0, s>>>(a);
  else
    k_rms_norm<T, W, VEC, N, false, false><<<grid, block, 0, s>>>(a);
  SO3_LAUNCH("rms_norm");
}

int backward_blocks(long long rows, int threads) {
  const bool warp = threads == 32;
  const long long want = warp ? (rows + kWarpRows - 1) / kWarpRows : rows;
  const int per_sm = warp ? 4 : std::max(1, std::min(8, 1024 / threads));
  return int(std::min<long long>(want, (long long)kSmCount * per_sm));
}

template <class T, class W, int VEC, int N>
void norm_backward(const so3lr_rms_norm_backward_args &a, float *partial, cudaStream_t s) {
  const int threads = row_threads(a.width, VEC * N);
  const int grid = backward_blocks(a.rows, threads);
  if (grid > 0) {
    if (threads == 32)
      k_rms_norm_backward<T, W, VEC, N, true>
          <<<grid, 32 * kWarpRows, kWarpRows * a.width * sizeof(float), s>>>(a, partial);
    else
      k_rms_norm_backward<T, W, VEC, N, false><<<grid, threads, 0, s>>>(a, partial);
    SO3_LAUNCH("rms_norm_backward");
  }
  k_column_sum<W><<<unsigned((a.width + 31) / 32), dim3(32, 32), 0, s>>>(grid, int(a.width), partial,
                                                                        static_cast<W *>(a.dweight));
  SO3_LAUNCH("column_sum");
}

template <class T, int VEC, int N>
void gate(const so3lr_gate_int8_args &a, cudaStream_t s) {
  const int threads = row_threads(a.hidden, VEC * N);
  if (threads == 32)
    k_gate_int8<T, VEC, N, true><<<unsigned((a.rows + kWarpRows - 1) / kWarpRows), 32 * kWarpRows, 0, s>>>(a);
  else
    k_gate_int8<T, VEC, N, false><<<unsigned(a.rows), threads, 0, s>>>(a);
  SO3_LAUNCH("gate_int8");
}

}  // namespace

void launch_rms_norm(const so3lr_rms_norm_args &a, cudaStream_t s) {
  by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    by_weight<T>(a.dtype, a.weight_dtype, [&](auto w) {
      using W = decltype(w);
      constexpr int V = 16 / sizeof(T);
      const int e = sizeof(T);
      const bool wide = a.width % V == 0 && aligned(a.x, a.x_stride, e, 16) &&
                        aligned(a.residual, a.residual_stride, e, 16) && aligned(a.s, a.s_stride, e, 16) &&
                        aligned(a.y, a.y_stride, e, 16) && aligned(a.codes, a.codes_stride, 1, V) &&
                        aligned(a.weight, 0, 1, 16);
      if (!wide)
        norm_forward<T, W, 1, kPerThread>(a, s);
      else
        norm_forward<T, W, V, kPerThread / V>(a, s);
    });
  });
}

long long rms_norm_backward_bytes(const so3lr_rms_norm_backward_args &a) {
  return (long long)backward_blocks(a.rows, row_threads(a.width, kPerThread)) * a.width * 4;
}

void launch_rms_norm_backward(const so3lr_rms_norm_backward_args &a, void *workspace, cudaStream_t s) {
  by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    by_weight<T>(a.dtype, a.weight_dtype, [&](auto w) {
      using W = decltype(w);
      constexpr int V = 16 / sizeof(T);
      const int e = sizeof(T);
      const bool wide = a.width % V == 0 && aligned(a.dy, a.dy_stride, e, 16) && aligned(a.s, a.s_stride, e, 16) &&
                        aligned(a.ds, a.ds_stride, e, 16) && aligned(a.dx, a.dx_stride, e, 16) &&
                        aligned(a.weight, 0, 1, 16);
      float *partial = static_cast<float *>(workspace);
      if (!wide)
        norm_backward<T, W, 1, kPerThread>(a, partial, s);
      else
        norm_backward<T, W, V, kPerThread / V>(a, partial, s);
    });
  });
}

void launch_gate_int8(const so3lr_gate_int8_args &a, cudaStream_t s) {
  by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / sizeof(T);
    const int e = sizeof(T);
    const bool wide = a.hidden % V == 0 && aligned(a.gu, a.gu_stride, e, 16) && aligned(a.codes, a.codes_stride, 1, V);
    // up to 32 elements per thread: 32768 columns in a block of 1,024 threads
    if (!wide)
      gate<T, 1, 32>(a, s);
    else if (a.hidden <= 1024 * kPerThread)
      gate<T, V, kPerThread / V>(a, s);
    else
      gate<T, V, 32 / V>(a, s);
  });
}

void launch_dequantize_int8(const so3lr_dequantize_int8_args &a, cudaStream_t s) {
  by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    const int e = sizeof(T);
    const bool wide = a.width % 8 == 0 && aligned(a.codes, a.codes_stride, 1, 8) && aligned(a.out, a.out_stride, e, 16);
    const long long total = a.rows * (wide ? a.width / 8 : a.width);
    const unsigned grid = unsigned(std::min<long long>((total + 255) / 256, kSmCount * 64));
    if (wide)
      k_dequantize_int8<T, 8><<<grid, 256, 0, s>>>(a);
    else
      k_dequantize_int8<T, 1><<<grid, 256, 0, s>>>(a);
    SO3_LAUNCH("dequantize_int8");
  });
}

}  // namespace so3lr_b200
