// Row kernels of the feed-forward layers: RMS norm with the residual's addition
// (forward, 8-bit output, backward), the 8-bit gate and the reading back of 8-bit
// rows. All are bound by HBM: every input element is read once into registers,
// every output written once; the row statistics are reduced between the two.
//
// A row belongs to one warp (up to 16 elements per lane, so that short rows need
// no block barrier) or to one block. A thread holds N chunks of VEC elements:
// 16-byte chunks where every row starts on a 16-byte boundary, single elements
// otherwise (odd widths, views). Eight elements a thread keep the registers low and
// so the bytes in flight high; sixteen only where a row would not fit otherwise.
#include "layers_common.cuh"
#include "model_host.hpp"
#include "tensor_core.cuh"

namespace so3lr_b200 {
namespace {

constexpr int kWarpRows = 8;     // rows of a block when a warp owns a row

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
  dependents_may_start();
  wait_for_predecessors();
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
        float sum[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] = to_float(cx[j].e[i]) + to_float(cr[j].e[i]);
        cx[j] = to_chunk<T, VEC>(sum);
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
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * team.size + team.t) * VEC;
    if (c < width) {
      float y[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        y[i] = v[j * VEC + i] * rstd * to_float(cw[j].e[i]);
        v[j * VEC + i] = y[i];
        if (QUANT) top = max_abs(top, y[i]);
      }
      if (!QUANT) store_chunk<T, VEC>(static_cast<T *>(a.y) + row * a.y_stride + c, to_chunk<T, VEC>(y));
    }
  }
  if (!QUANT) return;
  float inv;
  const float scale = row_scale(team.max(__float_as_uint(top) & 0x7fffffffu, slot_max), inv);
  if (team.t == 0) a.scales[row] = scale;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * team.size + team.t) * VEC;
    if (c < width)
      store_chunk<signed char, VEC>(a.codes + row * a.codes_stride + c, to_codes<VEC>(v + j * VEC, inv));
  }
}

// dx = rstd (a - xh mean(a xh)) + ds with a = dy w, xh = s rstd; each block also
// sums dy xh over its rows (a fixed set, in order) into one row of `partial`.
template <class T, class W, int VEC, int N, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 512 ? 2 : 1) k_rms_norm_backward(const so3lr_rms_norm_backward_args a, float *__restrict__ partial) {
  constexpr bool WARP = MAXT == 32 * kWarpRows;
  __shared__ float2 slot[2][32];
  extern __shared__ float column[];  // WARP: kWarpRows x width
  dependents_may_start();
  wait_for_predecessors();
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
        float out[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float xh = to_float(cs[j].e[i]) * rstd, d = to_float(cd[j].e[i]);
          dw[j * VEC + i] = fmaf(d, xh, dw[j * VEC + i]);
          float g = rstd * (d * to_float(cw[j].e[i]) - xh * mean);
          if (ds) g += to_float(ce[j].e[i]);
          out[i] = g;
        }
        store_chunk<T, VEC>(static_cast<T *>(a.dx) + row * a.dx_stride + c, to_chunk<T, VEC>(out));
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

// A ring of rows in shared memory, filled by bulk copies: what is in flight costs no
// registers, so a block that walks over rows keeps the memory system busy while it
// reduces and writes the current one. One block barrier after the last read of a
// stage, thread 0 may refill it.
struct RowRing {
  uint32_t bars, buffer, stage_bytes;
  int stages;
  unsigned char *mem;
  int *err;
  volatile int *abort_flag;

  __device__ RowRing(unsigned char *smem, uint32_t bytes, int nstages, int *error)
      : stage_bytes(bytes), stages(nstages), mem(smem + 128), err(error) {
    bars = tc::smem_u32(smem);
    buffer = bars + 128;
    abort_flag = reinterpret_cast<volatile int *>(smem + 120);
    if (threadIdx.x == 0) {
      for (int i = 0; i < stages; ++i) tc::mbar_init(bars + 8 * i, 1);
      *abort_flag = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
  }
  __device__ const unsigned char *stage(int i) const { return mem + (i % stages) * stage_bytes; }
  // waits for the i-th row of this block; after a wait that gave up (reported in *err) nothing waits again
  __device__ void wait(int i) const { tc::mbar_wait(bars + 8 * (i % stages), (i / stages) & 1, abort_flag, err, 7); }
  // thread 0: the copies of the i-th row
  __device__ uint32_t expect(int i, uint32_t bytes) const {
    tc::mbar_expect_tx(bars + 8 * (i % stages), bytes);
    return buffer + (i % stages) * stage_bytes;
  }
  __device__ uint32_t bar(int i) const { return bars + 8 * (i % stages); }
};
constexpr int kRingHeader = 128, kRingStages = 8;

// k_rms_norm_backward for rows on 16-byte boundaries that need a block: 16 elements a
// thread, rows through a ring. Bound by instruction issue before it is bound by HBM:
// the row's reduction costs each warp about a hundred instructions, so fewer and
// fuller warps are faster (8 elements a thread: 115 us at 16384 x 4096 bfloat16).
template <class T, class W>
__global__ void __launch_bounds__(512)
    k_rms_norm_backward_ring(const so3lr_rms_norm_backward_args a, float *__restrict__ partial, int stages, int *err) {
  constexpr int VEC = 16 / sizeof(T), N = 16 / VEC;
  __shared__ float2 slot[2][32];
  extern __shared__ __align__(128) unsigned char smem[];
  const int width = int(a.width), t = threadIdx.x, size = blockDim.x;
  const uint32_t row_bytes = width * sizeof(T), tensors = a.ds ? 3 : 2;
  dependents_may_start();
  const RowRing ring(smem, tensors * row_bytes, stages, err);
  wait_for_predecessors();
  const RowTeam<false> team;
  const int rows = a.rows > blockIdx.x ? int((a.rows - 1 - blockIdx.x) / gridDim.x) + 1 : 0;
  auto fetch = [&](int i) {
    const long long row = blockIdx.x + (long long)i * gridDim.x;
    const uint32_t dst = ring.expect(i, tensors * row_bytes);
    tc::bulk_load(dst, static_cast<const T *>(a.s) + row * a.s_stride, row_bytes, ring.bar(i));
    tc::bulk_load(dst + row_bytes, static_cast<const T *>(a.dy) + row * a.dy_stride, row_bytes, ring.bar(i));
    if (a.ds)
      tc::bulk_load(dst + 2 * row_bytes, static_cast<const T *>(a.ds) + row * a.ds_stride, row_bytes, ring.bar(i));
  };
  if (t == 0)
    for (int i = 0; i < min(stages, rows); ++i) fetch(i);
  Chunk<W, VEC> cw[N];
  float dw[16];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * size + t) * VEC;
    if (c < width) cw[j] = load_chunk<W, VEC>(static_cast<const W *>(a.weight) + c);
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[j * VEC + i] = 0.0f;
  }
  const float per = 1.0f / float(width);
  for (int k = 0; k < rows; ++k) {
    ring.wait(k);
    const T *s = reinterpret_cast<const T *>(ring.stage(k));
    Chunk<T, VEC> cs[N], cd[N], ce[N];
    float sq = 0.0f, dot = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * size + t) * VEC;
      if (c < width) {
        cs[j] = load_chunk<T, VEC>(s + c);
        cd[j] = load_chunk<T, VEC>(s + width + c);
        if (a.ds) ce[j] = load_chunk<T, VEC>(s + 2 * width + c);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float f = to_float(cs[j].e[i]);
          sq = fmaf(f, f, sq);
          dot = fmaf(f, to_float(cd[j].e[i]) * to_float(cw[j].e[i]), dot);
        }
      }
    }
    const float2 total = team.sum2(sq, dot, slot[k & 1]);  // a barrier: every thread has read the stage
    if (t == 0 && k + stages < rows && !*ring.abort_flag) fetch(k + stages);
    const float rstd = 1.0f / sqrtf(total.x * per + float(a.eps));
    const float back = -(total.y * rstd * per) * rstd * rstd;  // - mean(a xh) rstd^2, times s
    T *dx = static_cast<T *>(a.dx) + (blockIdx.x + (long long)k * gridDim.x) * a.dx_stride;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * size + t) * VEC;
      if (c < width) {
        float out[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float f = to_float(cs[j].e[i]), d = to_float(cd[j].e[i]);
          dw[j * VEC + i] = fmaf(d, f * rstd, dw[j * VEC + i]);
          const float rest = a.ds ? fmaf(f, back, to_float(ce[j].e[i])) : f * back;
          out[i] = fmaf(d * to_float(cw[j].e[i]), rstd, rest);
        }
        store_chunk<T, VEC>(dx + c, to_chunk<T, VEC>(out));
      }
    }
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * size + t) * VEC;
    if (c < width)
#pragma unroll
      for (int i = 0; i < VEC; ++i) partial[(size_t)blockIdx.x * width + c + i] = dw[j * VEC + i];
  }
}

// column sums of `partial` (nparts x width) in a fixed order: 32 columns per
// block, part k summed by thread row k % 32, then the 32 thread rows in order
template <class W>
__global__ void k_column_sum(int nparts, int width, const float *__restrict__ partial, W *__restrict__ out) {
  __shared__ float part[32][33];
  dependents_may_start();
  wait_for_predecessors();
  const int c = blockIdx.x * 32 + threadIdx.x;
  float total = 0.0f;
  if (c < width)
#pragma unroll 8
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

// 8-bit rows of silu(g) u
template <class T, int VEC, int N, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kWarpRows : 1024, VEC *N == 8 && !WARP ? 2 : 1)
    k_gate_int8(const so3lr_gate_int8_args a) {
  __shared__ uint32_t slot[32];
  dependents_may_start();
  wait_for_predecessors();
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
  float v[N * VEC], top = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * team.size + team.t) * VEC;
    if (c < hidden) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[j * VEC + i] = silu_f32(to_float(cg[j].e[i])) * to_float(cu[j].e[i]);
        top = max_abs(top, v[j * VEC + i]);
      }
    }
  }
  float inv;
  const float scale = row_scale(team.max(__float_as_uint(top) & 0x7fffffffu, slot), inv);
  if (team.t == 0) a.scales[row] = scale;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * team.size + team.t) * VEC;
    if (c < hidden)
      store_chunk<signed char, VEC>(a.codes + row * a.codes_stride + c, to_codes<VEC>(v + j * VEC, inv));
  }
}

// k_gate_int8 for many rows on 16-byte boundaries: PER elements a thread, rows through a ring
template <class T, int PER, int MAXT>
__global__ void __launch_bounds__(MAXT) k_gate_int8_ring(const so3lr_gate_int8_args a, int stages, int *err) {
  constexpr int VEC = 16 / sizeof(T), N = PER / VEC;
  __shared__ uint32_t slot[2][32];
  extern __shared__ __align__(128) unsigned char smem[];
  const int hidden = int(a.hidden), t = threadIdx.x, size = blockDim.x;
  const uint32_t row_bytes = 2 * hidden * sizeof(T);
  dependents_may_start();
  const RowRing ring(smem, row_bytes, stages, err);
  wait_for_predecessors();
  const RowTeam<false> team;
  const int rows = a.rows > blockIdx.x ? int((a.rows - 1 - blockIdx.x) / gridDim.x) + 1 : 0;
  auto fetch = [&](int i) {
    const long long row = blockIdx.x + (long long)i * gridDim.x;
    const uint32_t dst = ring.expect(i, row_bytes);
    tc::bulk_load(dst, static_cast<const T *>(a.gu) + row * a.gu_stride, row_bytes, ring.bar(i));
  };
  if (t == 0)
    for (int i = 0; i < min(stages, rows); ++i) fetch(i);
  for (int k = 0; k < rows; ++k) {
    ring.wait(k);
    const T *g = reinterpret_cast<const T *>(ring.stage(k)), *u = g + hidden;
    float v[PER], top = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * size + t) * VEC;
      if (c < hidden) {
        const Chunk<T, VEC> cg = load_chunk<T, VEC>(g + c), cu = load_chunk<T, VEC>(u + c);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          v[j * VEC + i] = silu_f32(to_float(cg.e[i])) * to_float(cu.e[i]);
          top = max_abs(top, v[j * VEC + i]);
        }
      }
    }
    float inv;
    const uint32_t bits = team.max(__float_as_uint(top) & 0x7fffffffu, slot[k & 1]);  // every thread has read the stage
    if (t == 0 && k + stages < rows && !*ring.abort_flag) fetch(k + stages);
    const float scale = row_scale(bits, inv);
    const long long row = blockIdx.x + (long long)k * gridDim.x;
    if (t == 0) a.scales[row] = scale;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * size + t) * VEC;
      if (c < hidden)
        store_chunk<signed char, VEC>(a.codes + row * a.codes_stride + c, to_codes<VEC>(v + j * VEC, inv));
    }
  }
}

template <class T, int VEC>
__global__ void k_dequantize_int8(const so3lr_dequantize_int8_args a) {
  dependents_may_start();
  wait_for_predecessors();
  const long long per_row = a.width / VEC, total = a.rows * per_row;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const long long row = total < (1LL << 31) ? uint32_t(i) / uint32_t(per_row) : i / per_row;
    const long long c = (i - row * per_row) * VEC;
    const Chunk<signed char, VEC> q = load_chunk<signed char, VEC>(a.codes + row * a.codes_stride + c);
    const float scale = a.scales[row];
    T *dst = static_cast<T *>(a.out) + row * a.out_stride + c;
    if (VEC == 16) {
      constexpr int kPer = 16 / sizeof(T);
#pragma unroll
      for (int j = 0; j < VEC; j += kPer) {
        float out[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k)
          out[k] = byte_to_float(reinterpret_cast<const uint32_t *>(&q)[(j + k) / 4] ^ 0x80808080u, (j + k) % 4) * scale;
        store_chunk<T, kPer>(dst + j, to_chunk<T, kPer>(out));
      }
    } else {
      dst[0] = from_float<T>(float(q.e[0]) * scale);
    }
  }
}

// ------------------------------------------------------------------ dispatch
bool aligned(const void *p, long long stride, int size, int bytes) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && (stride * size) % bytes == 0);
}

// Threads that hold a row of `width` elements, `per` of them each: a warp where one
// suffices, else a block of whole warps.
int row_threads(long long width, int per) { return int((width + 32LL * per - 1) / (32LL * per)) * 32; }
// Elements a thread holds: 8, or 16 where that keeps the row in one warp or in one block.
int per_thread(long long width) { return width <= 256 || (width > 512 && width <= 8192) ? 8 : 16; }

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
    launch(k_rms_norm<T, W, VEC, N, true, true>, grid, block, 0, s, a);
  else if (warp)
    launch(k_rms_norm<T, W, VEC, N, true, false>, grid, block, 0, s, a);
  else if (a.codes)
    launch(k_rms_norm<T, W, VEC, N, false, true>, grid, block, 0, s, a);
  else
    launch(k_rms_norm<T, W, VEC, N, false, false>, grid, block, 0, s, a);
}

// Blocks of a kernel that walks over rows
int walking_blocks(long long rows, int threads) {
  const bool warp = threads == 32;
  const long long want = warp ? (rows + kWarpRows - 1) / kWarpRows : rows;
  const int per_sm = warp ? 4 : std::max(1, std::min(8, 1024 / threads));
  return int(std::min<long long>(want, (long long)kSmCount * per_sm));
}

// Ring of a kernel that walks over rows: as many blocks an SM as its registers hold
// (`resident` threads), shared memory for up to kRingStages rows each. stages < 2: the
// row is too long.
struct RingPlan {
  int grid, stages, smem;
};
RingPlan ring_plan(long long rows, int threads, int resident, long long row_bytes) {
  const int per_sm = std::max(1, std::min(16, resident / threads));
  const long long room = 220 * 1024 / per_sm - 2048 - kRingHeader;  // 2 KB: static and reserved shared memory
  RingPlan p;
  p.grid = int(std::min<long long>(rows, (long long)kSmCount * per_sm));
  p.stages = int(std::min<long long>(kRingStages, room / row_bytes));
  p.smem = int(kRingHeader + p.stages * row_bytes);
  return p;
}
// The ring kernel's blocks, 0 where the direct loads serve: rows of a warp, unaligned
// rows, and rows too long for the ring
RingPlan backward_ring(const so3lr_rms_norm_backward_args &a) {
  const int e = a.dtype == SO3LR_FLOAT32 ? 4 : 2;
  const bool wide = a.width * e % 16 == 0 && aligned(a.dy, a.dy_stride, e, 16) && aligned(a.s, a.s_stride, e, 16) &&
                    aligned(a.ds, a.ds_stride, e, 16) && aligned(a.dx, a.dx_stride, e, 16) &&
                    aligned(a.weight, 0, 1, 16);
  if (!wide || a.width <= 512 || a.width > 8192) return RingPlan{0, 0, 0};
  const RingPlan p = ring_plan(a.rows, row_threads(a.width, 16), 512, 3 * a.width * e);
  return p.stages < 2 ? RingPlan{0, 0, 0} : p;
}
int backward_parts(const so3lr_rms_norm_backward_args &a) {
  const RingPlan r = backward_ring(a);
  return r.stages ? r.grid : walking_blocks(a.rows, row_threads(a.width, per_thread(a.width)));
}

template <class T, class W, int VEC, int N>
void norm_backward(const so3lr_rms_norm_backward_args &a, float *partial, int grid, cudaStream_t s) {
  const int threads = row_threads(a.width, VEC * N);
  if (threads == 32) {
    launch(k_rms_norm_backward<T, W, VEC, N, 32 * kWarpRows>, grid, 32 * kWarpRows,
           kWarpRows * a.width * sizeof(float), s, a, partial);
    return;
  }
  // rows of a block that do not go through the ring: unaligned ones, and those too long for it
  if constexpr (VEC == 1 && N == 8) {
    if (threads <= 512) {
      launch(k_rms_norm_backward<T, W, VEC, N, 512>, grid, threads, 0, s, a, partial);
      return;
    }
  }
  launch(k_rms_norm_backward<T, W, VEC, N, 1024>, grid, threads, 0, s, a, partial);
}
template <class T, class W>
void norm_backward_ring(const so3lr_rms_norm_backward_args &a, float *partial, const RingPlan &r, cudaStream_t s) {
  check_gave_up();
  const int threads = row_threads(a.width, 16);
  auto run = [&](auto fn) {
    allow_dynamic_smem(reinterpret_cast<const void *>(fn), 227 * 1024 - 1024);
    launch(fn, r.grid, threads, r.smem, s, a, partial, r.stages, gave_up_flag());
  };
  run(&k_rms_norm_backward_ring<T, W>);
}

template <class T, int VEC, int N>
void gate(const so3lr_gate_int8_args &a, cudaStream_t s) {
  const int threads = row_threads(a.hidden, VEC * N);
  if (threads == 32)
    launch(k_gate_int8<T, VEC, N, true>, unsigned((a.rows + kWarpRows - 1) / kWarpRows), 32 * kWarpRows, 0, s, a);
  else
    launch(k_gate_int8<T, VEC, N, false>, unsigned(a.rows), threads, 0, s, a);
}
int ring_per_thread(long long hidden) { return hidden <= 4096 ? 16 : 32; }
template <class T>
void gate_ring(const so3lr_gate_int8_args &a, const RingPlan &r, cudaStream_t s) {
  check_gave_up();
  const int threads = row_threads(a.hidden, ring_per_thread(a.hidden));
  auto run = [&](auto fn) {
    allow_dynamic_smem(reinterpret_cast<const void *>(fn), 227 * 1024 - 1024);
    launch(fn, r.grid, threads, r.smem, s, a, r.stages, gave_up_flag());
  };
  if (ring_per_thread(a.hidden) == 16)
    run(&k_gate_int8_ring<T, 16, 256>);
  else
    run(&k_gate_int8_ring<T, 32, 512>);
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
      if (per_thread(a.width) == 8)
        wide ? norm_forward<T, W, V, 8 / V>(a, s) : norm_forward<T, W, 1, 8>(a, s);
      else
        wide ? norm_forward<T, W, V, 16 / V>(a, s) : norm_forward<T, W, 1, 16>(a, s);
    });
  });
}

long long rms_norm_backward_bytes(const so3lr_rms_norm_backward_args &a) {
  return (long long)backward_parts(a) * a.width * 4;
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
      const RingPlan r = backward_ring(a);
      const int parts = backward_parts(a);
      if (parts > 0) {
        if (r.stages)
          norm_backward_ring<T, W>(a, partial, r, s);
        else if (per_thread(a.width) == 8)
          wide ? norm_backward<T, W, V, 8 / V>(a, partial, parts, s) : norm_backward<T, W, 1, 8>(a, partial, parts, s);
        else
          wide ? norm_backward<T, W, V, 16 / V>(a, partial, parts, s)
               : norm_backward<T, W, 1, 16>(a, partial, parts, s);
      }
      launch(k_column_sum<W>, unsigned((a.width + 31) / 32), dim3(32, 32), 0, s, parts, int(a.width), partial, static_cast<W *>(a.dweight));
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
    const int per = a.hidden > 16384 ? 32 : per_thread(a.hidden);
    // the ring where a block has several rows to walk over, and a row needs a block
    const RingPlan r = ring_plan(a.rows, row_threads(a.hidden, ring_per_thread(a.hidden)), 1024, 2 * a.hidden * e);
    if (wide && a.hidden > 512 && a.hidden <= 16384 && r.stages >= 2 && a.rows > 2 * r.grid)
      gate_ring<T>(a, r, s);
    else if (per == 32)
      wide ? gate<T, V, 32 / V>(a, s) : gate<T, 1, 32>(a, s);
    else if (per == 8)
      wide ? gate<T, V, 8 / V>(a, s) : gate<T, 1, 8>(a, s);
    else
      wide ? gate<T, V, 16 / V>(a, s) : gate<T, 1, 16>(a, s);
  });
}

void launch_dequantize_int8(const so3lr_dequantize_int8_args &a, cudaStream_t s) {
  by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    const int e = sizeof(T);
    const bool wide =
        a.width % 16 == 0 && aligned(a.codes, a.codes_stride, 1, 16) && aligned(a.out, a.out_stride, e, 16);
    const long long total = a.rows * (wide ? a.width / 16 : a.width);
    const unsigned grid = unsigned(std::min<long long>((total + 255) / 256, kSmCount * 64));
    if (wide)
      launch(k_dequantize_int8<T, 16>, grid, 256, 0, s, a);
    else
      launch(k_dequantize_int8<T, 1>, grid, 256, 0, s, a);
  });
}

}  // namespace so3lr_b200
