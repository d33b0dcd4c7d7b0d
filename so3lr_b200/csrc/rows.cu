// Row kernels of the feed-forward layers: RMS norm with the residual's addition
// (forward, 8-bit output, backward), the 8-bit gate and the reading back of 8-bit
// rows. All are bound by HBM: every input element is read once into registers,
// every output written once; the row statistics are reduced between the two.
//
// A row belongs to 8, 16 or 32 lanes of a warp (rows of up to 1024 elements: no block
// barrier) or to one block. A thread holds N chunks of VEC elements: 16-byte chunks,
// from the row's start where every row is on a 16-byte boundary, else from the first
// boundary in the row (odd widths, views: Span), and single elements where the
// tensors' rows lie differently. With 2-byte elements the kernels issue more than they
// load unless a thread has many elements: a row's reduction, its reciprocal root and
// addresses cost each thread about a hundred instructions, an element about ten. Long
// 8-bit rows and gradients walk over their rows with a ring of copies in flight.
//
// Measured, 33.5 M bfloat16 elements, float32 weights, rows of 256 / 4096 / 1003: norm with
// residual 6.5 / 6.5 / 4.5 TB/s (a copy: 6.5), 8-bit norm without 3.4 / 3.7 / 1.8 (bfloat16
// weights 3.7 / 3.7 / 2.2), gradient with ds 5.5 / 5.3 / 3.8, 8-bit gate 5.9 / 6.3 / 4.0,
// reading back 5.9 / 6.2 / 3.9. The 8-bit norm issues 21 instructions an element at 0.8 of
// the issue rate, the gradient 29 at 0.6.
#include "row_team.cuh"

namespace so3lr_b200 {
namespace {

// The scale of a row of s w rstd from the bits of max|s w|; `inv` takes v and ve, the row's
// s w, to codes. inv is 127 / max|s w|, which overflows below 2^-121: rows of less than 2^-100
// are lifted by 2^64 first.
// Against y / scale the codes' quotient carries the roundings of s w, the reciprocal and
// rstd, a few float32 units: a y that near a tie may fall on its other side.
template <int COUNT>
__device__ __forceinline__ float norm_scale(float mean_square, uint32_t top_bits, float &inv, float (&v)[COUNT],
                                            float &ve) {
  const float rstd = rsqrtf(mean_square), top = __uint_as_float(top_bits);
  const float y = top * rstd;
  float scale = y * (1.0f / 127.0f);
  inv = __fdividef(1.0f, scale) * rstd;
  // One test for all that row_scale looks at and for rows to lift; a NaN fails it. With
  // row_scale on every row's path 131072 x 256 bfloat16 takes 30.5 us, so 29.8.
  if (!(fminf(top * 0x1p-26f, scale) >= 0x1p-126f && y <= 3.4028234e38f)) {
    scale = row_scale(__float_as_uint(y) & 0x7fffffffu, inv);
    if (inv != 0.0f) {
      if (top < 0x1p-100f) {
        inv *= 0x1p-64f;
#pragma unroll
        for (int i = 0; i < COUNT; ++i) v[i] *= 0x1p64f;
        ve *= 0x1p64f;
      }
      inv *= rstd;
    }
  }
  return scale;
}

// y = s w rstd, s = x + residual as stored. QUANT: y goes to 8 bits with the row's scale.
template <class T, class W, int VEC, int N, int LANES, bool QUANT, bool SHIFT>
__global__ void __launch_bounds__(LANES ? kTeamThreads : 1024)
    k_rms_norm(const so3lr_rms_norm_args a, const float inv_width, const float eps) {
  __shared__ float slot[32];
  __shared__ uint32_t slot_max[32];
  dependents_may_start();
  wait_for_predecessors();
  const RowTeam<LANES> team;
  bool live;
  const long long row = team_row<LANES>(a.rows, live);
  const int width = int(a.width);
  const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
  const T *r = a.residual ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
  T *s = static_cast<T *>(a.s) + row * a.s_stride;
  const W *w = static_cast<const W *>(a.weight);
  const Span<SHIFT, VEC> span(x, width, team.t);

  Chunk<T, VEC> cx[N], cr[N];
  Chunk<W, VEC> cw[N];
  T ex{}, er{};
  W ew{};
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = span.at(j * team.size + team.t);
    if (span.holds(c)) {
      cx[j] = load_chunk<T, VEC>(x + c);
      if (r) cr[j] = load_chunk<T, VEC>(r + c);
      cw[j] = load_apart<SHIFT, W, VEC>(w + c);
    }
  }
  if (span.edge >= 0) {
    ex = x[span.edge];
    if (r) er = r[span.edge];
    ew = w[span.edge];
  }
  float v[N * VEC], ve = 0.0f, sq = 0.0f, top = 0.0f;  // v: s, or (QUANT) s w
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = span.at(j * team.size + team.t);
    if (span.holds(c)) {
      if (r) {
        // the stream is kept in the element type, and the norm is of what is kept
        float sum[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] = to_float(cx[j].e[i]) + to_float(cr[j].e[i]);
        cx[j] = to_chunk<T, VEC>(sum);
        if (live) store_chunk<T, VEC>(s + c, cx[j]);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[j * VEC + i] = to_float(cx[j].e[i]);
        sq = fmaf(v[j * VEC + i], v[j * VEC + i], sq);
        if (QUANT) {
          v[j * VEC + i] *= to_float(cw[j].e[i]);
          top = max_abs(top, v[j * VEC + i]);
        }
      }
    }
  }
  if (span.edge >= 0) {
    if (r) {
      ex = from_float<T>(to_float(ex) + to_float(er));
      if (live) s[span.edge] = ex;
    }
    ve = to_float(ex);
    sq = fmaf(ve, ve, sq);
    if (QUANT) {
      ve *= to_float(ew);
      top = max_abs(top, ve);
    }
  }
  if (QUANT) {  // the largest y is that of s w: both statistics in one reduction
    uint32_t bits = __float_as_uint(top) & 0x7fffffffu;
    const float sum = team.sum_and_max(sq, bits, slot, slot_max);
    float inv;
    const float scale = norm_scale(fmaf(sum, inv_width, eps), bits, inv, v, ve);
    if (!live) return;
    if (team.t == 0) a.scales[row] = scale;
    signed char *codes = a.codes + row * a.codes_stride;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = span.at(j * team.size + team.t);
      if (span.holds(c)) store_apart<SHIFT, signed char, VEC>(codes + c, to_codes<VEC>(v + j * VEC, inv));
    }
    if (span.edge >= 0) codes[span.edge] = to_codes<1>(&ve, inv).e[0];
    return;
  }
  const float rstd = rsqrtf(fmaf(team.sum(sq, slot), inv_width, eps));
  if (!live) return;
  T *out = static_cast<T *>(a.y) + row * a.y_stride;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = span.at(j * team.size + team.t);
    if (span.holds(c)) {
      float y[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) y[i] = v[j * VEC + i] * rstd * to_float(cw[j].e[i]);
      store_chunk<T, VEC>(out + c, to_chunk<T, VEC>(y));
    }
  }
  if (span.edge >= 0) out[span.edge] = from_float<T>(ve * rstd * to_float(ew));
}

// dx = rstd (a - xh mean(a xh)) + ds with a = dy w, xh = s rstd; each block also
// sums dy xh over its rows (a fixed set, in order) into one row of `partial`.
template <class T, class W, int VEC, int N, int LANES, int MAXT, bool SHIFT>
__global__ void __launch_bounds__(MAXT, MAXT == 512 ? 2 : VEC *N == 8 && LANES ? 4 : LANES ? 2 : 1)
    k_rms_norm_backward(const so3lr_rms_norm_backward_args a, float *__restrict__ partial, const float inv_width,
                        const float eps) {
  __shared__ float2 slot[2][32];
  extern __shared__ float column[];  // LANES: teams x width
  dependents_may_start();
  wait_for_predecessors();
  const RowTeam<LANES> team;
  const int width = int(a.width);
  constexpr int kTeams = LANES ? kTeamThreads / (LANES ? LANES : 1) : 1;
  const int team_id = LANES ? threadIdx.x / (LANES ? LANES : 1) : 0;
  // SHIFT: the grid's rows a step are a multiple of 8, so that a team's rows share their span
  const Span<SHIFT, VEC> span(static_cast<const T *>(a.s) + ((long long)blockIdx.x * kTeams + team_id) * a.s_stride,
                              width, team.t);
  const W *w = static_cast<const W *>(a.weight);
  Chunk<W, VEC> cw[N];
  float dw[N * VEC], we = span.edge >= 0 ? to_float(w[span.edge]) : 0.0f, dwe = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = span.at(j * team.size + team.t);
    if (span.holds(c)) cw[j] = load_apart<SHIFT, W, VEC>(w + c);
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[j * VEC + i] = 0.0f;
  }
  int parity = 0;
  // whole blocks walk together; a team past the last row adds nothing
  for (long long first = (long long)blockIdx.x * kTeams; first < a.rows; first += (long long)gridDim.x * kTeams) {
    const bool live = first + team_id < a.rows;
    const long long row = live || SHIFT ? first + team_id : a.rows - 1;
    const T *s = static_cast<const T *>(a.s) + row * a.s_stride;
    const T *dy = static_cast<const T *>(a.dy) + row * a.dy_stride;
    const T *ds = a.ds ? static_cast<const T *>(a.ds) + row * a.ds_stride : nullptr;
    Chunk<T, VEC> cs[N], cd[N], ce[N];
    T es{}, ed{}, ee{};
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = span.at(j * team.size + team.t);
      if (SHIFT) cs[j] = cd[j] = ce[j] = Chunk<T, VEC>{};
      if ((live || !SHIFT) && span.holds(c)) {  // the last row again, or (another span) none
        cs[j] = load_chunk<T, VEC>(s + c);
        cd[j] = load_chunk<T, VEC>(dy + c);
        if (ds) ce[j] = load_chunk<T, VEC>(ds + c);
      }
    }
    const bool edge = live && span.edge >= 0;
    if (edge) {
      es = s[span.edge];
      ed = dy[span.edge];
      if (ds) ee = ds[span.edge];
    }
    float sq = 0.0f, dot = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (span.holds(span.at(j * team.size + team.t))) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float f = to_float(cs[j].e[i]);
          sq = fmaf(f, f, sq);
          dot = fmaf(f, to_float(cd[j].e[i]) * to_float(cw[j].e[i]), dot);
        }
      }
    }
    if (SHIFT) {
      sq = fmaf(to_float(es), to_float(es), sq);
      dot = fmaf(to_float(es), to_float(ed) * we, dot);
    }
    const float2 total = team.sum2(sq, dot, slot[parity]);
    parity ^= 1;
    if (!live) continue;
    const float rstd = rsqrtf(fmaf(total.x, inv_width, eps));
    const float back = -(total.y * rstd * inv_width) * rstd * rstd;  // - mean(a xh) rstd^2, times s
    T *dx = static_cast<T *>(a.dx) + row * a.dx_stride;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = span.at(j * team.size + team.t);
      if (span.holds(c)) {
        float out[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float f = to_float(cs[j].e[i]), d = to_float(cd[j].e[i]);
          dw[j * VEC + i] = fmaf(d, f * rstd, dw[j * VEC + i]);
          const float rest = ds ? fmaf(f, back, to_float(ce[j].e[i])) : f * back;
          out[i] = fmaf(d * to_float(cw[j].e[i]), rstd, rest);
        }
        store_chunk<T, VEC>(dx + c, to_chunk<T, VEC>(out));
      }
    }
    if (edge) {
      const float f = to_float(es), d = to_float(ed);
      dwe = fmaf(d, f * rstd, dwe);
      dx[span.edge] = from_float<T>(fmaf(d * we, rstd, ds ? fmaf(f, back, to_float(ee)) : f * back));
    }
  }
  float *sums = LANES ? column + team_id * width : partial + (size_t)blockIdx.x * width;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = span.at(j * team.size + team.t);
    if (span.holds(c))
#pragma unroll
      for (int i = 0; i < VEC; ++i) sums[c + i] = dw[j * VEC + i];
  }
  if (span.edge >= 0) sums[span.edge] = dwe;
  if (!LANES) return;
  __syncthreads();
  for (int c = threadIdx.x; c < width; c += blockDim.x) {
    float total = 0.0f;
#pragma unroll
    for (int k = 0; k < kTeams; ++k) total += column[k * width + c];
    partial[(size_t)blockIdx.x * width + c] = total;
  }
}

// k_rms_norm to 8 bits for many rows of 2-byte elements on 16-byte boundaries: 16
// elements a thread, rows through a ring, the weight in registers
template <class T, class W>
__global__ void __launch_bounds__(512)
    k_rms_norm_int8_ring(const so3lr_rms_norm_args a, int stages, const WaitLimit limit, const float inv_width,
                         const float eps) {
  constexpr int VEC = 16 / sizeof(T), N = 16 / VEC;
  __shared__ float slot[2][32];
  __shared__ uint32_t slot_max[2][32];
  extern __shared__ __align__(128) unsigned char smem[];
  const int width = int(a.width), t = threadIdx.x, size = blockDim.x;
  const uint32_t row_bytes = width * sizeof(T), tensors = a.residual ? 2 : 1;
  dependents_may_start();
  const RowRing ring(smem, tensors * row_bytes, stages, limit);
  wait_for_predecessors();
  const RowTeam<0> team;
  const int rows = a.rows > blockIdx.x ? int((a.rows - 1 - blockIdx.x) / gridDim.x) + 1 : 0;
  auto fetch = [&](int i) {
    const long long row = blockIdx.x + (long long)i * gridDim.x;
    const uint32_t dst = ring.expect(i, tensors * row_bytes);
    tc::bulk_load(dst, static_cast<const T *>(a.x) + row * a.x_stride, row_bytes, ring.bar(i));
    if (a.residual)
      tc::bulk_load(dst + row_bytes, static_cast<const T *>(a.residual) + row * a.residual_stride, row_bytes,
                    ring.bar(i));
  };
  if (t == 0)
    for (int i = 0; i < min(stages, rows); ++i) fetch(i);
  Chunk<W, VEC> cw[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * size + t) * VEC;
    if (c < width) cw[j] = load_chunk<W, VEC>(static_cast<const W *>(a.weight) + c);
  }
  int k = 0;
  for (; k < rows; ++k) {
    ring.wait(k);
    const T *x = reinterpret_cast<const T *>(ring.stage(k));
    const long long row = blockIdx.x + (long long)k * gridDim.x;
    float v[16], sq = 0.0f, top = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * size + t) * VEC;
      if (c < width) {
        Chunk<T, VEC> cx = load_chunk<T, VEC>(x + c);
        if (a.residual) {
          const Chunk<T, VEC> cr = load_chunk<T, VEC>(x + width + c);
          float sum[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) sum[i] = to_float(cx.e[i]) + to_float(cr.e[i]);
          cx = to_chunk<T, VEC>(sum);
          store_chunk<T, VEC>(static_cast<T *>(a.s) + row * a.s_stride + c, cx);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float f = to_float(cx.e[i]);
          sq = fmaf(f, f, sq);
          v[j * VEC + i] = f * to_float(cw[j].e[i]);
          top = max_abs(top, v[j * VEC + i]);
        }
      }
    }
    uint32_t bits = __float_as_uint(top) & 0x7fffffffu;
    const float sum = team.sum_and_max(sq, bits, slot[k & 1], slot_max[k & 1]);  // a barrier, as below
    if (ring.gave_up(k)) break;
    if (t == 0 && k + stages < rows) fetch(k + stages);
    float inv, none = 0.0f;
    const float scale = norm_scale(fmaf(sum, inv_width, eps), bits, inv, v, none);
    if (t == 0) a.scales[row] = scale;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * size + t) * VEC;
      if (c < width)
        store_chunk<signed char, VEC>(a.codes + row * a.codes_stride + c, to_codes<VEC>(v + j * VEC, inv));
    }
  }
  if (t == 0) ring.settle(k, rows);
}

// k_rms_norm_backward for rows on 16-byte boundaries that need a block: 16 elements a
// thread, rows through a ring. Bound by instruction issue before it is bound by HBM:
// the row's reduction costs each warp about a hundred instructions, so fewer and
// fuller warps are faster (16384 x 4096 bfloat16: 91 us, 115 with 8 elements a thread).
template <class T, class W>
__global__ void __launch_bounds__(512)
    k_rms_norm_backward_ring(const so3lr_rms_norm_backward_args a, float *__restrict__ partial, int stages,
                             const WaitLimit limit, const float inv_width, const float eps) {
  constexpr int VEC = 16 / sizeof(T), N = 16 / VEC;
  __shared__ float2 slot[2][32];
  extern __shared__ __align__(128) unsigned char smem[];
  const int width = int(a.width), t = threadIdx.x, size = blockDim.x;
  const uint32_t row_bytes = width * sizeof(T), tensors = a.ds ? 3 : 2;
  dependents_may_start();
  const RowRing ring(smem, tensors * row_bytes, stages, limit);
  wait_for_predecessors();
  const RowTeam<0> team;
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
  int k = 0;
  for (; k < rows; ++k) {
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
    if (ring.gave_up(k)) break;
    if (t == 0 && k + stages < rows) fetch(k + stages);
    const float rstd = rsqrtf(fmaf(total.x, inv_width, eps));
    const float back = -(total.y * rstd * inv_width) * rstd * rstd;  // - mean(a xh) rstd^2, times s
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
  if (t == 0) ring.settle(k, rows);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * size + t) * VEC;
    if (c < width)
#pragma unroll
      for (int i = 0; i < VEC; ++i) partial[(size_t)blockIdx.x * width + c + i] = dw[j * VEC + i];
  }
}

// column sums of `partial` (nparts x width) in a fixed order: 32 columns per
// block, part k summed by thread row k % 32, then the 32 thread rows in order. No
// __restrict__: the kernel that writes `partial` may still run when this one starts.
template <class W>
__global__ void k_column_sum(int nparts, int width, const float *partial, W *out) {
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
template <class T, int VEC, int N, int LANES, bool SHIFT>
__global__ void __launch_bounds__(LANES ? kTeamThreads : 1024) k_gate_int8(const so3lr_gate_int8_args a) {
  __shared__ uint32_t slot[32];
  dependents_may_start();
  wait_for_predecessors();
  const RowTeam<LANES> team;
  bool live;
  const long long row = team_row<LANES>(a.rows, live);
  const int hidden = int(a.hidden);
  const T *g = static_cast<const T *>(a.gu) + row * a.gu_stride, *u = g + hidden;
  const Span<SHIFT, VEC> span(g, hidden, team.t);
  Chunk<T, VEC> cg[N], cu[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = span.at(j * team.size + team.t);
    if (span.holds(c)) {
      cg[j] = load_chunk<T, VEC>(g + c);
      cu[j] = load_apart<SHIFT, T, VEC>(u + c);
    }
  }
  float v[N * VEC], ve = 0.0f, top = 0.0f;
  if (span.edge >= 0) {
    ve = silu_f32(to_float(g[span.edge])) * to_float(u[span.edge]);
    top = max_abs(top, ve);
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (span.holds(span.at(j * team.size + team.t))) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[j * VEC + i] = silu_f32(to_float(cg[j].e[i])) * to_float(cu[j].e[i]);
        top = max_abs(top, v[j * VEC + i]);
      }
    }
  }
  float inv;
  const float scale = row_scale(team.max(__float_as_uint(top) & 0x7fffffffu, slot), inv);
  if (!live) return;
  if (team.t == 0) a.scales[row] = scale;
  signed char *codes = a.codes + row * a.codes_stride;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = span.at(j * team.size + team.t);
    if (span.holds(c)) store_apart<SHIFT, signed char, VEC>(codes + c, to_codes<VEC>(v + j * VEC, inv));
  }
  if (span.edge >= 0) codes[span.edge] = to_codes<1>(&ve, inv).e[0];
}

// WIDE: 16 codes a thread, rows of both on 16-byte boundaries. Otherwise a 16-byte chunk
// of the result, counted from the boundary before its row, from single codes.
template <class T, bool WIDE>
__global__ void k_dequantize_int8(const so3lr_dequantize_int8_args a) {
  dependents_may_start();
  wait_for_predecessors();
  constexpr int kPer = 16 / sizeof(T), VEC = WIDE ? 16 : kPer;
  const int width = int(a.width);
  const long long per_row = WIDE ? a.width / VEC : (a.width + 2 * VEC - 2) / VEC, total = a.rows * per_row;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const long long row = total < (1LL << 31) ? uint32_t(i) / uint32_t(per_row) : i / per_row;
    const signed char *codes = a.codes + row * a.codes_stride;
    T *out = static_cast<T *>(a.out) + row * a.out_stride;
    const int shift = WIDE ? 0 : int(reinterpret_cast<uintptr_t>(out) % 16 / sizeof(T));
    const int c = int(i - row * per_row) * VEC - shift;
    if (c >= width) continue;
    const float scale = a.scales[row];
    if (!WIDE && (c < 0 || c + VEC > width)) {
      for (int k = max(c, 0); k < min(c + VEC, width); ++k) out[k] = from_float<T>(float(codes[k]) * scale);
      continue;
    }
    const Chunk<signed char, VEC> q = load_apart<!WIDE, signed char, VEC>(codes + c);
#pragma unroll
    for (int j = 0; j < VEC; j += kPer) {
      float f[kPer];
#pragma unroll
      for (int k = 0; k < kPer; ++k)
        f[k] = WIDE ? byte_to_float(reinterpret_cast<const uint32_t *>(&q)[(j + k) / 4] ^ 0x80808080u, (j + k) % 4) * scale
                    : float(q.e[j + k]) * scale;
      store_chunk<T, kPer>(out + c + j, to_chunk<T, kPer>(f));
    }
  }
}

// ------------------------------------------------------------------ dispatch
Path backward_path(const so3lr_rms_norm_backward_args &a) {
  RowTensors t{a.dtype == SO3LR_FLOAT32 ? 4 : 2};
  t.add(a.dy, a.dy_stride);
  t.add(a.s, a.s_stride);
  t.add(a.ds, a.ds_stride);
  t.add(a.dx, a.dx_stride);
  return t.path(a.width, aligned(a.weight, 0, 1, 16));
}
Hold backward_hold(const so3lr_rms_norm_backward_args &a, Path path) {
  return hold(a.width, path, a.dtype == SO3LR_FLOAT32 ? 4 : 2, kNormBack);
}
// The ring kernel's blocks, no stages where the direct loads serve: rows of a warp,
// rows off the boundaries, and rows too long for the ring
RingPlan backward_ring(const so3lr_rms_norm_backward_args &a) {
  if (backward_path(a) != kWide || a.width <= 512 || a.width > 8192) return RingPlan{0, 0, 0};
  // two rows deep: float32, 2048 wide, 4.6 TB/s of inputs in four blocks an SM, 3.4 in three, three deep
  // (8192 wide, the longest: 96 KB a row, two of them in one)
  return ring_plan(a.rows, row_threads(a.width, 16), 512, 2, 3 * a.width * (a.dtype == SO3LR_FLOAT32 ? 4 : 2));
}
int backward_parts(const so3lr_rms_norm_backward_args &a) {
  const RingPlan r = backward_ring(a);
  if (r.stages) return r.grid;
  const Path path = backward_path(a);
  const Hold h = backward_hold(a, path);
  const int blocks = walking_blocks(h, a.rows, a.width);
  return path == kShifted && h.lanes == 0 ? (blocks + 7) / 8 * 8 : blocks;
}

template <class T, class W, Path PATH>
void norm_backward(const so3lr_rms_norm_backward_args &a, float *partial, int grid, cudaStream_t s) {
  constexpr int V = chunk_of(PATH, sizeof(T));
  constexpr bool SHIFT = PATH == kShifted;
  const Hold h = backward_hold(a, PATH);
  by_hold<PATH, sizeof(T), kNormBack>(h, [&](auto lanes, auto per) {
    constexpr int L = decltype(lanes)::value, P = decltype(per)::value, N = P / V;
    const float inv = 1.0f / float(a.width), eps = float(a.eps);
    if constexpr (L != 0) {
      launch(k_rms_norm_backward<T, W, V, N, L, kTeamThreads, SHIFT>, grid, kTeamThreads,
             kTeamThreads / L * a.width * sizeof(float), s, a, partial, inv, eps);
    } else {
      // rows that start elsewhere than on 16-byte boundaries, and those too long for the ring
      const int threads = row_threads(a.width, P);
      if constexpr (P == 8) {
        if (PATH == kShifted || threads <= 512) {  // shifted: up to 4096 elements, see hold()
          launch(k_rms_norm_backward<T, W, V, N, 0, 512, SHIFT>, grid, threads, 0, s, a, partial, inv, eps);
          return;
        }
      }
      if constexpr (PATH != kShifted || P != 8)
        launch(k_rms_norm_backward<T, W, V, N, 0, 1024, SHIFT>, grid, threads, 0, s, a, partial, inv, eps);
    }
  });
}
template <class T, class W>
void norm_int8_ring(const so3lr_rms_norm_args &a, const RingPlan &r, cudaStream_t s) {
  allow_dynamic_smem(reinterpret_cast<const void *>(&k_rms_norm_int8_ring<T, W>), 227 * 1024 - 1024);
  launch(k_rms_norm_int8_ring<T, W>, r.grid, row_threads(a.width, 16), r.smem, s, a, r.stages, wait_limit(),
         1.0f / float(a.width), float(a.eps));
}
template <class T, class W>
void norm_backward_ring(const so3lr_rms_norm_backward_args &a, float *partial, const RingPlan &r, cudaStream_t s) {
  allow_dynamic_smem(reinterpret_cast<const void *>(&k_rms_norm_backward_ring<T, W>), 227 * 1024 - 1024);
  launch(k_rms_norm_backward_ring<T, W>, r.grid, row_threads(a.width, 16), r.smem, s, a, partial, r.stages,
         wait_limit(), 1.0f / float(a.width), float(a.eps));
}

}  // namespace

void launch_rms_norm(const so3lr_rms_norm_args &a, cudaStream_t s) {
  by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    by_weight<T>(a.dtype, a.weight_dtype, [&](auto w) {
      using W = decltype(w);
      constexpr int V = 16 / sizeof(T);
      RowTensors t{int(sizeof(T))};
      t.add(a.x, a.x_stride);
      t.add(a.residual, a.residual_stride);
      t.add(a.s, a.s_stride);
      t.add(a.y, a.y_stride);
      const Path chosen = t.path(a.width, aligned(a.codes, a.codes_stride, 1, V) && aligned(a.weight, 0, 1, 16));
      // The ring for many long rows of 2-byte elements (2048: 26 us, 31 without; 904: 34, 39; 768: 40, 33;
      // with a residual 2048: 42, 47; 768: 52, 66; float32 2048: 18, 15), two rows deep and twice the
      // blocks that fit, which evens out their ends (2048: 28 us with those that fit).
      if constexpr (sizeof(T) == 2) {
        const RingPlan r =
            ring_plan(a.rows, row_threads(a.width, 16), 2048, 2, (a.residual ? 2 : 1) * a.width * sizeof(T));
        if (chosen == kWide && a.codes && a.width > (a.residual ? 512 : 896) && a.width <= 8192 && r.stages >= 2 &&
            a.rows > 2 * r.grid) {
          norm_int8_ring<T, W>(a, r, s);
          return;
        }
      }
      by_path(chosen, [&](auto path) {
        constexpr Path PATH = decltype(path)::value;
        constexpr int VEC = chunk_of(PATH, sizeof(T));
        auto run = [&](auto op) {
          constexpr RowOp OP = decltype(op)::value;
          const Hold h = hold(a.width, PATH, sizeof(T), OP);
          by_hold<PATH, sizeof(T), OP>(h, [&](auto lanes, auto per) {
            constexpr int L = decltype(lanes)::value, N = decltype(per)::value / VEC;
            launch(k_rms_norm<T, W, VEC, N, L, OP == kNorm8, PATH == kShifted>, team_grid(h, a.rows),
                   team_block(h, a.width), 0, s, a, 1.0f / float(a.width), float(a.eps));
          });
        };
        if (a.codes)
          run(std::integral_constant<RowOp, kNorm8>{});
        else
          run(std::integral_constant<RowOp, kNorm>{});
      });
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
      float *partial = static_cast<float *>(workspace);
      const RingPlan r = backward_ring(a);
      const int parts = backward_parts(a);
      if (parts > 0) {
        if (r.stages)
          norm_backward_ring<T, W>(a, partial, r, s);
        else
          by_path(backward_path(a), [&](auto path) {
            norm_backward<T, W, decltype(path)::value>(a, partial, parts, s);
          });
      }
      launch(k_column_sum<W>, unsigned((a.width + 31) / 32), dim3(32, 32), 0, s, parts, int(a.width), partial,
             static_cast<W *>(a.dweight));
    });
  });
}

void launch_gate_int8(const so3lr_gate_int8_args &a, cudaStream_t s) {
  by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / sizeof(T);
    const int e = sizeof(T);
    const bool wide = a.hidden % V == 0 && aligned(a.gu, a.gu_stride, e, 16) && aligned(a.codes, a.codes_stride, 1, V);
    const Path chosen = wide ? kWide : a.hidden <= 16384 ? kShifted : kScalar;
    const Hold h = hold(a.hidden, chosen, e, kGate8);
    by_path(chosen, [&](auto path) {
      constexpr Path PATH = decltype(path)::value;
      constexpr int VEC = chunk_of(PATH, sizeof(T));
      by_hold<PATH, sizeof(T), kGate8>(h, [&](auto lanes, auto per) {
        constexpr int L = decltype(lanes)::value, N = decltype(per)::value / VEC;
        launch(k_gate_int8<T, VEC, N, L, PATH == kShifted>, team_grid(h, a.rows), team_block(h, a.hidden), 0, s, a);
      });
    });
  });
}

void launch_dequantize_int8(const so3lr_dequantize_int8_args &a, cudaStream_t s) {
  by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    const int e = sizeof(T);
    const bool wide =
        a.width % 16 == 0 && aligned(a.codes, a.codes_stride, 1, 16) && aligned(a.out, a.out_stride, e, 16);
    const long long total = a.rows * (wide ? a.width / 16 : (a.width + 2 * (16 / e) - 2) / (16 / e));
    const unsigned grid = unsigned(std::min<long long>((total + 255) / 256, kSmCount * 64));
    launch(wide ? &k_dequantize_int8<T, true> : &k_dequantize_int8<T, false>, grid, 256, 0, s, a);
  });
}

}  // namespace so3lr_b200
