// The norms on both sides of a block's boundary, in one pass over the rows:
//
//   s = residual scale + gate norm(x) weight,  y = norm(s) next_weight
//   norm(v) = v / sqrt(mean(v^2) + eps), of s as stored
//
// and their gradients: with rx, rs the reciprocal roots, xh = x rx, sh = s rs,
//
//   g = rs (dy next_weight - sh mean(dy next_weight sh)) + ds,  dnext_weight = sum dy sh
//   dresidual = g scale,  dscale = sum g residual,  dgate = g xh weight
//   q = g gate,  dweight = sum q xh,  dx = rx (q weight - xh mean(q weight xh))
//
// Bound by HBM: the forward pass moves 5 elements for each of a row, the backward pass 9;
// apart, the two norms, the gate and the sums would move 11 and 20. A row belongs to
// lanes of a warp or to a block as in rows.cu. The backward kernels walk over their rows
// and hold the three column sums; each block writes one row of them, and k_column_sums
// adds those in order.
//
// Measured, 33.5 M elements with gate and scale, forward and backward (TB/s): bfloat16 rows of
// 256 5.9 and 5.0, of 1024 5.8 and 5.2, of 4096 6.0 and 4.6, of 1003 4.0 and 3.3, of 16384 4.1 and
// 1.8; float32 rows (half as many) 6.5 and 6.0, 6.5 and 6.1, 6.2 and 5.3, 5.7 and 5.3, 4.7 and 3.0.
// Rows off the boundaries past 4096 elements go one element at a time in the backward pass: bfloat16 of
// 8191 2.2 and 0.75 (803 us), float32 3.5 and 1.5.
// With 2-byte elements a row's two reductions, about 50 instructions a thread, and one block of
// 512 threads an SM (the column sums fill the registers) hold the backward pass back.
#include "pairs.cuh"
#include "row_team.cuh"

namespace so3lr_b200 {
namespace {

// 1 / sqrt(a): a Newton step on the hardware's root, within a unit. The root's error is the whole
// row's, and shows in how many elements of the stream round to the other side.
__device__ __forceinline__ float inverse_root(float a) {
  const float y = rsqrtf(a), e = fmaf(-a * y, y, 1.0f);
  return fabsf(e) < 1.0f ? fmaf(0.5f * y, e, y) : y;  // 0, infinities and NaN as they are
}

template <class T>
struct SandwichRow {  // pointers to one row
  const T *x, *residual, *gate;
  T *s, *y;
  __device__ SandwichRow(const so3lr_sandwich_norm_args &a, long long row)
      : x(static_cast<const T *>(a.x) + row * a.x_stride),
        residual(static_cast<const T *>(a.residual) + row * a.residual_stride),
        gate(a.gate ? static_cast<const T *>(a.gate) + row * a.gate_stride : nullptr),
        s(static_cast<T *>(a.s) + row * a.s_stride),
        y(static_cast<T *>(a.y) + row * a.y_stride) {}
};

// The stream as it is kept, and its squares: residual scale + gate (x rx weight), rounded.
template <class T, class W, int VEC>
__device__ __forceinline__ Chunk<T, VEC> stream_of(const Chunk<T, VEC> &cx, const Chunk<T, VEC> &cr,
                                                   const Chunk<T, VEC> &cg, const Chunk<W, VEC> &cw,
                                                   const Chunk<W, VEC> &cc, float rx, typename Floats<VEC>::V &squares) {
  using F = Floats<VEC>;
  using V = typename F::V;
  const F x = floats_of(cx), r = floats_of(cr), g = floats_of(cg), w = floats_of(cw), scale = floats_of(cc);
  F s;
#pragma unroll
  for (int i = 0; i < F::kCount; ++i) s.v[i] = madd(g.v[i], x.v[i] * V(rx) * w.v[i], r.v[i] * scale.v[i]);
  const Chunk<T, VEC> kept = chunk_of_floats<T, VEC>(s);
  s = floats_of(kept);
#pragma unroll
  for (int i = 0; i < F::kCount; ++i) squares = madd(s.v[i], s.v[i], squares);
  return kept;
}
template <class T, class W, int VEC>
__device__ __forceinline__ Chunk<T, VEC> normed(const Chunk<T, VEC> &cs, const Chunk<W, VEC> &cn, float rs) {
  using F = Floats<VEC>;
  const F s = floats_of(cs), next = floats_of(cn);
  F y;
#pragma unroll
  for (int i = 0; i < F::kCount; ++i) y.v[i] = s.v[i] * typename F::V(rs) * next.v[i];
  return chunk_of_floats<T, VEC>(y);
}

template <class T, class W, int VEC, int N, int LANES, bool SHIFT>
__global__ void __launch_bounds__(LANES ? kTeamThreads : 1024)
    k_sandwich(const so3lr_sandwich_norm_args a, const float inv_width, const float eps) {
  __shared__ float slot[2][32];
  dependents_may_start();
  wait_for_predecessors();
  const RowTeam<LANES> team;
  bool live;
  const SandwichRow<T> row(a, team_row<LANES>(a.rows, live));
  const W *w = static_cast<const W *>(a.weight), *next = static_cast<const W *>(a.next_weight),
          *scale = static_cast<const W *>(a.residual_scale);
  const Span<SHIFT, VEC> span(row.x, int(a.width), team.t);
  Chunk<T, VEC> cx[N], cr[N], cg[N];
  T ex{}, er{}, eg = from_float<T>(1.0f);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = span.at(j * team.size + team.t);
    cg[j] = ones<T, VEC>();
    if (span.holds(c)) {
      cx[j] = load_chunk<T, VEC>(row.x + c);
      cr[j] = load_chunk<T, VEC>(row.residual + c);
      if (row.gate) cg[j] = load_chunk<T, VEC>(row.gate + c);
    }
  }
  if (span.edge >= 0) {
    ex = row.x[span.edge];
    er = row.residual[span.edge];
    if (row.gate) eg = row.gate[span.edge];
  }
  using F = Floats<VEC>;
  using V = typename F::V;
  V squares(0.0f);
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (span.holds(span.at(j * team.size + team.t))) {
      const F x = floats_of(cx[j]);
#pragma unroll
      for (int i = 0; i < F::kCount; ++i) squares = madd(x.v[i], x.v[i], squares);
    }
  float sq = fmaf(to_float(ex), to_float(ex), total(squares));
  const float rx = inverse_root(fmaf(team.sum(sq, slot[0]), inv_width, eps));
  // what is kept of the stream is rounded, and the second norm is of what is kept
  squares = V(0.0f);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = span.at(j * team.size + team.t);
    if (span.holds(c)) {
      cx[j] = stream_of(cx[j], cr[j], cg[j], load_apart<SHIFT, W, VEC>(w + c),
                        scale ? load_apart<SHIFT, W, VEC>(scale + c) : ones<W, VEC>(), rx, squares);
      if (live) store_chunk<T, VEC>(row.s + c, cx[j]);
    }
  }
  sq = total(squares);
  if (span.edge >= 0) {
    const int c = span.edge;
    float one = 0.0f;
    ex = stream_of(Chunk<T, 1>{{ex}}, Chunk<T, 1>{{er}}, Chunk<T, 1>{{eg}}, Chunk<W, 1>{{w[c]}},
                   Chunk<W, 1>{{scale ? scale[c] : from_float<W>(1.0f)}}, rx, one)
             .e[0];
    if (live) row.s[c] = ex;
    sq += one;
  }
  const float rs = inverse_root(fmaf(team.sum(sq, slot[1]), inv_width, eps));
  if (!live) return;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = span.at(j * team.size + team.t);
    if (span.holds(c)) store_chunk<T, VEC>(row.y + c, normed(cx[j], load_apart<SHIFT, W, VEC>(next + c), rs));
  }
  if (span.edge >= 0) row.y[span.edge] = from_float<T>(to_float(ex) * rs * to_float(next[span.edge]));
}

template <class T>
struct SandwichBackRow {
  const T *dy, *ds, *s, *x, *residual, *gate;
  T *dx, *dresidual, *dgate;
  __device__ SandwichBackRow(const so3lr_sandwich_norm_backward_args &a, long long row)
      : dy(static_cast<const T *>(a.dy) + row * a.dy_stride),
        ds(a.ds ? static_cast<const T *>(a.ds) + row * a.ds_stride : nullptr),
        s(static_cast<const T *>(a.s) + row * a.s_stride),
        x(static_cast<const T *>(a.x) + row * a.x_stride),
        residual(a.residual_scale ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr),
        gate(a.gate ? static_cast<const T *>(a.gate) + row * a.gate_stride : nullptr),
        dx(static_cast<T *>(a.dx) + row * a.dx_stride),
        dresidual(static_cast<T *>(a.dresidual) + row * a.dresidual_stride),
        dgate(a.gate ? static_cast<T *>(a.dgate) + row * a.dgate_stride : nullptr) {}
};
// The gradient's elements (V: a float or a pair), all in float32. The row's first statistics give
// g and what follows from it; its last one, sum(a x), is there after them.
template <class V>
__device__ __forceinline__ void add_squares(const V &x, const V &s, const V &dy, const V &next, V (&sums)[3]) {
  sums[0] = madd(x, x, sums[0]);
  sums[1] = madd(s, s, sums[1]);
  sums[2] = madd(s, dy * next, sums[2]);
}
template <class V>
struct SandwichElement {
  V dres, dgate, a;
  // adds to the column sums of q xh, dy sh and g residual, and to the row's of a x
  __device__ __forceinline__ SandwichElement(const V &x, const V &s, const V &dy, const V &ds, const V &r,
                                             const V &gate, const V &w, const V &next, const V &scale, float rx,
                                             float rs, float back, V &sum_w, V &sum_next, V &sum_scale, V &row_sum) {
    const V g = madd(dy * next, V(rs), madd(s, V(back), ds)), xh = x * V(rx), q = g * gate;
    dres = g * scale;
    dgate = g * (xh * w);
    a = q * w;
    sum_w = madd(q, xh, sum_w);
    sum_next = madd(dy, s * V(rs), sum_next);
    sum_scale = madd(g, r, sum_scale);
    row_sum = madd(a, x, row_sum);
  }
};
// dx from a and the row's last statistic
template <class T, int VEC>
__device__ __forceinline__ Chunk<T, VEC> dx_of(const Floats<VEC> &a, const Chunk<T, VEC> &cx, float rx, float back_x) {
  using F = Floats<VEC>;
  using V = typename F::V;
  const F x = floats_of(cx);
  F dx;
#pragma unroll
  for (int i = 0; i < F::kCount; ++i) dx.v[i] = madd(a.v[i], V(rx), x.v[i] * V(back_x));
  return chunk_of_floats<T, VEC>(dx);
}

template <int VEC>
__device__ __forceinline__ void write_floats(float *p, const Floats<VEC> &f) {
  const Chunk<float, VEC> c = chunk_of_floats<float, VEC>(f);
#pragma unroll
  for (int i = 0; i < VEC; ++i) p[i] = c.e[i];
}

// Rows in registers, 8 or 16 elements a thread.
template <class T, class W, int VEC, int N, int LANES, bool SHIFT>
__global__ void __launch_bounds__(LANES ? kTeamThreads : 512, LANES && VEC *N == 8 ? 2 : 1)
    k_sandwich_backward(const so3lr_sandwich_norm_backward_args a, float *partial, const float inv_width,
                        const float eps) {
  __shared__ float2 slot2[32];
  __shared__ float slot[2][32];
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
  const W *w = static_cast<const W *>(a.weight), *next = static_cast<const W *>(a.next_weight),
          *scale = static_cast<const W *>(a.residual_scale);
  using F = Floats<VEC>;
  using V = typename F::V;
  F sums[3][N];
  float edge_sums[3] = {};
#pragma unroll
  for (int k = 0; k < 3; ++k)
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int i = 0; i < F::kCount; ++i) sums[k][j].v[i] = V(0.0f);
  // whole blocks walk together; a team past the last row adds nothing
  for (long long first = (long long)blockIdx.x * kTeams; first < a.rows; first += (long long)gridDim.x * kTeams) {
    const bool live = first + team_id < a.rows;
    const SandwichBackRow<T> row(a, live ? first + team_id : a.rows - 1);
    Chunk<T, VEC> cs[N], cd[N], ce[N], cx[N], cr[N], cg[N];
    T es{}, ed{}, ee{}, ex{}, er{}, eg = from_float<T>(1.0f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = span.at(j * team.size + team.t);
      cs[j] = cd[j] = ce[j] = cx[j] = cr[j] = Chunk<T, VEC>{};
      cg[j] = ones<T, VEC>();
      if (live && span.holds(c)) {
        cs[j] = load_chunk<T, VEC>(row.s + c);
        cd[j] = load_chunk<T, VEC>(row.dy + c);
        cx[j] = load_chunk<T, VEC>(row.x + c);
        if (row.ds) ce[j] = load_chunk<T, VEC>(row.ds + c);
        if (row.residual) cr[j] = load_chunk<T, VEC>(row.residual + c);
        if (row.gate) cg[j] = load_chunk<T, VEC>(row.gate + c);
      }
    }
    const bool edge = live && span.edge >= 0;
    if (edge) {
      es = row.s[span.edge];
      ed = row.dy[span.edge];
      ex = row.x[span.edge];
      if (row.ds) ee = row.ds[span.edge];
      if (row.residual) er = row.residual[span.edge];
      if (row.gate) eg = row.gate[span.edge];
    }
    V squares[3] = {V(0.0f), V(0.0f), V(0.0f)};
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = span.at(j * team.size + team.t);
      if (span.holds(c)) {
        const F x = floats_of(cx[j]), s = floats_of(cs[j]), dy = floats_of(cd[j]),
                n = floats_of(load_apart<SHIFT, W, VEC>(next + c));
#pragma unroll
        for (int i = 0; i < F::kCount; ++i) add_squares(x.v[i], s.v[i], dy.v[i], n.v[i], squares);
      }
    }
    float three[3] = {total(squares[0]), total(squares[1]), total(squares[2])};
    if (edge) add_squares(to_float(ex), to_float(es), to_float(ed), to_float(next[span.edge]), three);
    const float3 all = team.sum3(three[0], three[1], three[2], slot[0], slot2);
    const float rx = inverse_root(fmaf(all.x, inv_width, eps)), rs = inverse_root(fmaf(all.y, inv_width, eps));
    const float back = -(all.z * rs * inv_width) * rs * rs;
    F av[N];
    V row_sum(0.0f);
    float ae = 0.0f, last = 0.0f;
    if (live) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = span.at(j * team.size + team.t);
        if (span.holds(c)) {
          const F x = floats_of(cx[j]), s = floats_of(cs[j]), dy = floats_of(cd[j]), ds = floats_of(ce[j]),
                  r = floats_of(cr[j]), g = floats_of(cg[j]), wf = floats_of(load_apart<SHIFT, W, VEC>(w + c)),
                  n = floats_of(load_apart<SHIFT, W, VEC>(next + c)),
                  f = floats_of(scale ? load_apart<SHIFT, W, VEC>(scale + c) : ones<W, VEC>());
          F dres, dgate;
#pragma unroll
          for (int i = 0; i < F::kCount; ++i) {
            const SandwichElement<V> e(x.v[i], s.v[i], dy.v[i], ds.v[i], r.v[i], g.v[i], wf.v[i], n.v[i], f.v[i], rx, rs,
                                       back, sums[0][j].v[i], sums[1][j].v[i], sums[2][j].v[i], row_sum);
            dres.v[i] = e.dres;
            dgate.v[i] = e.dgate;
            av[j].v[i] = e.a;
          }
          store_chunk<T, VEC>(row.dresidual + c, chunk_of_floats<T, VEC>(dres));
          if (row.dgate) store_chunk<T, VEC>(row.dgate + c, chunk_of_floats<T, VEC>(dgate));
        }
      }
      last = total(row_sum);
    }
    if (edge) {
      const int c = span.edge;
      const SandwichElement<float> e(to_float(ex), to_float(es), to_float(ed), to_float(ee), to_float(er), to_float(eg),
                                     to_float(w[c]), to_float(next[c]), scale ? to_float(scale[c]) : 1.0f, rx, rs, back,
                                     edge_sums[0], edge_sums[1], edge_sums[2], last);
      row.dresidual[c] = from_float<T>(e.dres);
      if (row.dgate) row.dgate[c] = from_float<T>(e.dgate);
      ae = e.a;
    }
    const float back_x = -(team.sum(last, slot[1]) * rx * inv_width) * rx * rx;
    if (!live) continue;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = span.at(j * team.size + team.t);
      if (span.holds(c)) store_chunk<T, VEC>(row.dx + c, dx_of(av[j], cx[j], rx, back_x));
    }
    if (edge) row.dx[span.edge] = from_float<T>(fmaf(ae, rx, to_float(ex) * back_x));
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    float *mine = partial + ((size_t)blockIdx.x * 3 + k) * width;
    float *out = LANES ? column + team_id * width : mine;
    if (LANES) __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = span.at(j * team.size + team.t);
      if (span.holds(c)) write_floats(out + c, sums[k][j]);
    }
    if (span.edge >= 0) out[span.edge] = edge_sums[k];
    if (!LANES) continue;
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += blockDim.x) {
      float total = 0.0f;
#pragma unroll
      for (int t = 0; t < kTeams; ++t) total += column[t * width + c];
      mine[c] = total;
    }
  }
}

// Sums over a block of up to 16 warps, the same value to every thread; `slot` starts as zeros.
// The warps' parts are added by twos in every warp: each thread adding all 16 would cost a row of 8
// elements a thread a tenth of its instructions.
template <int K>
__device__ __forceinline__ void block_sums(float (&v)[K], float (*slot)[16]) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = RowTeam<0>::add(v[k]);
    if ((threadIdx.x & 31) == 0) slot[k][threadIdx.x >> 5] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = slot[k][threadIdx.x & 15];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
}

// k_sandwich for many long rows on 16-byte boundaries: rows through a ring, weights in
// registers. The stream's statistics need the first norm's, so a row goes through two block
// barriers; the copies of the next ones run on meanwhile.
template <class T, class W, int PER>
__global__ void __launch_bounds__(512, PER == 8 ? 2 : 1)
    k_sandwich_ring(const so3lr_sandwich_norm_args a, int stages, const WaitLimit limit, const float inv_width,
                    const float eps) {
  constexpr int VEC = 16 / sizeof(T), N = PER / VEC;
  using F = Floats<VEC>;
  using V = typename F::V;
  __shared__ __align__(16) float slot[2][16];
  extern __shared__ __align__(128) unsigned char smem[];
  const int width = int(a.width), t = threadIdx.x, size = blockDim.x;
  const uint32_t row_bytes = width * sizeof(T), tensors = a.gate ? 3 : 2;
  dependents_may_start();
  const RowRing ring(smem, tensors * row_bytes, stages, limit);
  wait_for_predecessors();
  if (t < 32) slot[t / 16][t % 16] = 0.0f;
  __syncthreads();
  const int rows = a.rows > blockIdx.x ? int((a.rows - 1 - blockIdx.x) / gridDim.x) + 1 : 0;
  auto fetch = [&](int i) {
    const long long row = blockIdx.x + (long long)i * gridDim.x;
    const uint32_t dst = ring.expect(i, tensors * row_bytes), bar = ring.bar(i);
    tc::bulk_load(dst, static_cast<const T *>(a.x) + row * a.x_stride, row_bytes, bar);
    tc::bulk_load(dst + row_bytes, static_cast<const T *>(a.residual) + row * a.residual_stride, row_bytes, bar);
    if (a.gate) tc::bulk_load(dst + 2 * row_bytes, static_cast<const T *>(a.gate) + row * a.gate_stride, row_bytes, bar);
  };
  if (t == 0)
    for (int i = 0; i < min(stages, rows); ++i) fetch(i);
  Chunk<W, VEC> cw[N], cn[N], cc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * size + t) * VEC;
    cc[j] = ones<W, VEC>();
    if (c < width) {
      cw[j] = load_chunk<W, VEC>(static_cast<const W *>(a.weight) + c);
      cn[j] = load_chunk<W, VEC>(static_cast<const W *>(a.next_weight) + c);
      if (a.residual_scale) cc[j] = load_chunk<W, VEC>(static_cast<const W *>(a.residual_scale) + c);
    }
  }
  int k = 0;
  for (; k < rows; ++k) {
    ring.wait(k);
    const T *x = reinterpret_cast<const T *>(ring.stage(k));
    const long long row = blockIdx.x + (long long)k * gridDim.x;
    Chunk<T, VEC> cx[N];
    V squares(0.0f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * size + t) * VEC;
      if (c < width) {
        cx[j] = load_chunk<T, VEC>(x + c);
        const F f = floats_of(cx[j]);
#pragma unroll
        for (int i = 0; i < F::kCount; ++i) squares = madd(f.v[i], f.v[i], squares);
      }
    }
    float sq[1] = {total(squares)};
    block_sums(sq, &slot[0]);
    const float rx = inverse_root(fmaf(sq[0], inv_width, eps));
    if (ring.gave_up(k)) break;
    squares = V(0.0f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * size + t) * VEC;
      if (c < width) {
        const Chunk<T, VEC> cg = a.gate ? load_chunk<T, VEC>(x + 2 * width + c) : ones<T, VEC>();
        cx[j] = stream_of(cx[j], load_chunk<T, VEC>(x + width + c), cg, cw[j], cc[j], rx, squares);
        store_chunk<T, VEC>(static_cast<T *>(a.s) + row * a.s_stride + c, cx[j]);
      }
    }
    sq[0] = total(squares);
    block_sums(sq, &slot[1]);
    const float rs = inverse_root(fmaf(sq[0], inv_width, eps));
    if (t == 0 && k + stages < rows) fetch(k + stages);  // every thread has read the stage
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * size + t) * VEC;
      if (c < width) store_chunk<T, VEC>(static_cast<T *>(a.y) + row * a.y_stride + c, normed(cx[j], cn[j], rs));
    }
  }
  if (t == 0) ring.settle(k, rows);
}

// k_sandwich_backward for rows on 16-byte boundaries that need a block, through a ring
template <class T, class W, int PER>
__global__ void __launch_bounds__(512)
    k_sandwich_backward_ring(const so3lr_sandwich_norm_backward_args a, float *partial, int stages,
                             const WaitLimit limit, const float inv_width, const float eps) {
  constexpr int VEC = 16 / sizeof(T), N = PER / VEC;
  using F = Floats<VEC>;
  using V = typename F::V;
  __shared__ __align__(16) float slot[4][16];
  extern __shared__ __align__(128) unsigned char smem[];
  const int width = int(a.width), t = threadIdx.x, size = blockDim.x;
  const uint32_t row_bytes = width * sizeof(T);
  // where each tensor of a row lies in its stage: s, dy, x, then those that there are
  const int ds_at = 3, gate_at = ds_at + (a.ds ? 1 : 0), residual_at = gate_at + (a.gate ? 1 : 0),
            tensors = residual_at + (a.residual_scale ? 1 : 0);
  dependents_may_start();
  const RowRing ring(smem, tensors * row_bytes, stages, limit);
  wait_for_predecessors();
  if (t < 64) slot[t / 16][t % 16] = 0.0f;
  __syncthreads();
  const int rows = a.rows > blockIdx.x ? int((a.rows - 1 - blockIdx.x) / gridDim.x) + 1 : 0;
  auto fetch = [&](int i) {
    const long long row = blockIdx.x + (long long)i * gridDim.x;
    const uint32_t dst = ring.expect(i, tensors * row_bytes), bar = ring.bar(i);
    auto copy = [&](const void *from, long long stride, int at) {
      tc::bulk_load(dst + at * row_bytes, static_cast<const T *>(from) + row * stride, row_bytes, bar);
    };
    copy(a.s, a.s_stride, 0);
    copy(a.dy, a.dy_stride, 1);
    copy(a.x, a.x_stride, 2);
    if (a.ds) copy(a.ds, a.ds_stride, ds_at);
    if (a.gate) copy(a.gate, a.gate_stride, gate_at);
    if (a.residual_scale) copy(a.residual, a.residual_stride, residual_at);
  };
  if (t == 0)
    for (int i = 0; i < min(stages, rows); ++i) fetch(i);
  Chunk<W, VEC> cw[N], cn[N], cc[N];
  F sums[3][N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * size + t) * VEC;
    cc[j] = ones<W, VEC>();
#pragma unroll
    for (int i = 0; i < F::kCount; ++i) sums[0][j].v[i] = sums[1][j].v[i] = sums[2][j].v[i] = V(0.0f);
    if (c < width) {
      cw[j] = load_chunk<W, VEC>(static_cast<const W *>(a.weight) + c);
      cn[j] = load_chunk<W, VEC>(static_cast<const W *>(a.next_weight) + c);
      if (a.residual_scale) cc[j] = load_chunk<W, VEC>(static_cast<const W *>(a.residual_scale) + c);
    }
  }
  int k = 0;
  for (; k < rows; ++k) {
    ring.wait(k);
    const T *stage = reinterpret_cast<const T *>(ring.stage(k));
    const SandwichBackRow<T> row(a, blockIdx.x + (long long)k * gridDim.x);
    Chunk<T, VEC> cs[N], cd[N], cx[N];
    V squares[3] = {V(0.0f), V(0.0f), V(0.0f)};
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * size + t) * VEC;
      if (c < width) {
        cs[j] = load_chunk<T, VEC>(stage + c);
        cd[j] = load_chunk<T, VEC>(stage + width + c);
        cx[j] = load_chunk<T, VEC>(stage + 2 * width + c);
        const F x = floats_of(cx[j]), s = floats_of(cs[j]), dy = floats_of(cd[j]), n = floats_of(cn[j]);
#pragma unroll
        for (int i = 0; i < F::kCount; ++i) add_squares(x.v[i], s.v[i], dy.v[i], n.v[i], squares);
      }
    }
    float first[3] = {total(squares[0]), total(squares[1]), total(squares[2])};
    block_sums(first, &slot[0]);
    if (ring.gave_up(k)) break;
    const float rx = inverse_root(fmaf(first[0], inv_width, eps)), rs = inverse_root(fmaf(first[1], inv_width, eps));
    const float back = -(first[2] * rs * inv_width) * rs * rs;
    F av[N];
    V row_sum(0.0f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * size + t) * VEC;
      if (c < width) {
        const F x = floats_of(cx[j]), s = floats_of(cs[j]), dy = floats_of(cd[j]),
                ds = floats_of(a.ds ? load_chunk<T, VEC>(stage + ds_at * width + c) : Chunk<T, VEC>{}),
                g = floats_of(a.gate ? load_chunk<T, VEC>(stage + gate_at * width + c) : ones<T, VEC>()),
                r = floats_of(a.residual_scale ? load_chunk<T, VEC>(stage + residual_at * width + c) : Chunk<T, VEC>{}),
                w = floats_of(cw[j]), n = floats_of(cn[j]), f = floats_of(cc[j]);
        F dres, dgate;
#pragma unroll
        for (int i = 0; i < F::kCount; ++i) {
          const SandwichElement<V> e(x.v[i], s.v[i], dy.v[i], ds.v[i], r.v[i], g.v[i], w.v[i], n.v[i], f.v[i], rx, rs,
                                     back, sums[0][j].v[i], sums[1][j].v[i], sums[2][j].v[i], row_sum);
          dres.v[i] = e.dres;
          dgate.v[i] = e.dgate;
          av[j].v[i] = e.a;
        }
        store_chunk<T, VEC>(row.dresidual + c, chunk_of_floats<T, VEC>(dres));
        if (a.gate) store_chunk<T, VEC>(row.dgate + c, chunk_of_floats<T, VEC>(dgate));
      }
    }
    float last[1] = {total(row_sum)};
    block_sums(last, &slot[3]);
    const float back_x = -(last[0] * rx * inv_width) * rx * rx;
    if (t == 0 && k + stages < rows) fetch(k + stages);  // every thread has read the stage
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * size + t) * VEC;
      if (c < width) store_chunk<T, VEC>(row.dx + c, dx_of(av[j], cx[j], rx, back_x));
    }
  }
  if (t == 0) ring.settle(k, rows);
#pragma unroll
  for (int q = 0; q < 3; ++q)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * size + t) * VEC;
      if (c < width) write_floats(partial + ((size_t)blockIdx.x * 3 + q) * width + c, sums[q][j]);
    }
}

// Any row, a block each, VEC elements at a time: elements are read again for each statistic
// (from L2, mostly), the column sums stand in shared memory, each thread's own.
template <class T, class W, int VEC>
__global__ void __launch_bounds__(512) k_sandwich_backward_long(const so3lr_sandwich_norm_backward_args a,
                                                                float *partial, const float inv_width,
                                                                const float eps) {
  __shared__ __align__(16) float slot[4][16];
  extern __shared__ __align__(16) float column[];  // 3 x width
  dependents_may_start();
  const int width = int(a.width), t = threadIdx.x, step = blockDim.x * VEC;
  if (t < 64) slot[t / 16][t % 16] = 0.0f;
  for (int c = t; c < 3 * width; c += blockDim.x) column[c] = 0.0f;
  __syncthreads();
  wait_for_predecessors();
  const W *w = static_cast<const W *>(a.weight), *next = static_cast<const W *>(a.next_weight),
          *scale = static_cast<const W *>(a.residual_scale);
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const SandwichBackRow<T> row(a, r);
    float first[3] = {};  // sums of x^2, s^2, s dy next
#pragma unroll 2
    for (int c = t * VEC; c < width; c += step) {
      const Chunk<T, VEC> cx = load_chunk<T, VEC>(row.x + c), cs = load_chunk<T, VEC>(row.s + c),
                          cd = load_chunk<T, VEC>(row.dy + c);
      const Chunk<W, VEC> cn = load_chunk<W, VEC>(next + c);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        add_squares(to_float(cx.e[i]), to_float(cs.e[i]), to_float(cd.e[i]), to_float(cn.e[i]), first);
      }
    }
    block_sums(first, &slot[0]);
    const float rx = inverse_root(fmaf(first[0], inv_width, eps)), rs = inverse_root(fmaf(first[1], inv_width, eps));
    const float back = -(first[2] * rs * inv_width) * rs * rs;
    // f(c, i, the element) over the row
    auto elements = [&](auto f) {
      for (int c = t * VEC; c < width; c += step) {
        const Chunk<T, VEC> cx = load_chunk<T, VEC>(row.x + c), cs = load_chunk<T, VEC>(row.s + c),
                            cd = load_chunk<T, VEC>(row.dy + c);
        const Chunk<W, VEC> cw = load_chunk<W, VEC>(w + c), cn = load_chunk<W, VEC>(next + c);
        Chunk<T, VEC> ce{}, cr{}, cg{};
        Chunk<W, VEC> cc{};
        if (row.ds) ce = load_chunk<T, VEC>(row.ds + c);
        if (row.residual) cr = load_chunk<T, VEC>(row.residual + c);
        if (row.gate) cg = load_chunk<T, VEC>(row.gate + c);
        if (scale) cc = load_chunk<W, VEC>(scale + c);
        auto element = [&](int i, float &sum_w, float &sum_next, float &sum_scale, float &row_sum) {
          return SandwichElement<float>(to_float(cx.e[i]), to_float(cs.e[i]), to_float(cd.e[i]), to_float(ce.e[i]),
                                        to_float(cr.e[i]), row.gate ? to_float(cg.e[i]) : 1.0f, to_float(cw.e[i]),
                                        to_float(cn.e[i]), scale ? to_float(cc.e[i]) : 1.0f, rx, rs, back, sum_w,
                                        sum_next, sum_scale, row_sum);
        };
        f(c, cx, element);
      }
    };
    float last[1] = {};
    elements([&](int c, const Chunk<T, VEC> &cx, auto element) {
      float dres[VEC], dgate[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const SandwichElement<float> e =
            element(i, column[c + i], column[width + c + i], column[2 * width + c + i], last[0]);
        dres[i] = e.dres;
        dgate[i] = e.dgate;
      }
      store_chunk<T, VEC>(row.dresidual + c, to_chunk<T, VEC>(dres));
      if (row.dgate) store_chunk<T, VEC>(row.dgate + c, to_chunk<T, VEC>(dgate));
    });
    block_sums(last, &slot[3]);
    const float back_x = -(last[0] * rx * inv_width) * rx * rx;
    elements([&](int c, const Chunk<T, VEC> &cx, auto element) {
      float dx[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float none[4] = {};
        dx[i] = fmaf(element(i, none[0], none[1], none[2], none[3]).a, rx, to_float(cx.e[i]) * back_x);
      }
      store_chunk<T, VEC>(row.dx + c, to_chunk<T, VEC>(dx));
    });
  }
  for (int c = t; c < 3 * width; c += blockDim.x) partial[(size_t)blockIdx.x * 3 * width + c] = column[c];
}

// Column sums of `partial` (nparts x 3 x width) in a fixed order, one output for each y of the grid
template <class W>
struct Sums {
  W *out[3];
};
template <class W>
__global__ void k_column_sums(int nparts, int width, const float *partial, const Sums<W> sums) {
  __shared__ float part[32][33];
  dependents_may_start();
  wait_for_predecessors();
  const int c = blockIdx.x * 32 + threadIdx.x;
  float total = 0.0f;
  if (c < width)
#pragma unroll 8
    for (int k = threadIdx.y; k < nparts; k += 32) total += partial[((size_t)k * 3 + blockIdx.y) * width + c];
  part[threadIdx.y][threadIdx.x] = total;
  __syncthreads();
  if (threadIdx.y == 0 && c < width) {
    total = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; ++k) total += part[k][threadIdx.x];
    sums.out[blockIdx.y][c] = from_float<W>(total);
  }
}

// -------------------------------------------------------------------- dispatch
// How a row is held, lanes of a warp (0: a block) and elements a thread. The backward pass
// holds rows of up to 4096 elements; per = 0: longer ones.
constexpr Hold sandwich_hold(long long width, Path path, int size, bool backward) {
  if (path != kScalar) {
    // rows off the boundaries: their edges take up to 2 (16 / size - 1) threads
    if (width <= 64 && (path == kWide || size == 4)) return {8, 8};
    if (width <= 128) return {16, 8};
  }
  if (width <= 512) return {32, width <= 256 ? 8 : 16};
  if (backward && width > 4096) return {0, 0};
  return {0, width <= 8192 ? 8 : 16};
}
// The rings take rows on the boundaries from these widths on, up to what a ring of two holds (us, 33.5
// M elements, in registers and through the ring). Forward, bfloat16 512: 52 and 61, 768: 65 and 59,
// 4096: 83 and 56; float32 (half as many) 1024: 51 and 59, 4096: 55 and 58, 8192: 71 and 58. Backward,
// bfloat16 512: 132 and 121, 4096: 188 and 132; float32 2048: 104 and 110, 4096: 121 and 114.
constexpr bool ring_takes(long long width, int size, bool backward) {
  return width > (backward ? (size == 2 ? 256 : 2048) : (size == 2 ? 512 : 4096)) && width <= 8192;
}
// Whether a call reaches the kernels that hold a row so: the widths are those at which
// sandwich_hold or ring_takes changes, each the widest of its kind.
constexpr bool held_so(Path path, int size, bool backward, int lanes, int per) {
  for (const int width : {64, 128, 256, 512, 2048, 4096, 8192, 16384}) {
    if (backward && path == kWide && ring_takes(width, size, true)) continue;
    const Hold h = sandwich_hold(width, path, size, backward);
    if (h.lanes == lanes && h.per == per) return true;
  }
  return false;
}
// f(std::integral_constant lanes, std::integral_constant per) for h; kernels are compiled for those
// that a call reaches
template <Path PATH, int SIZE, bool BACKWARD, class F>
void by_sandwich_hold(const Hold &h, F &&f) {
  bool found = false;
  auto lanes_per = [&](auto lanes, auto per) {
    if constexpr (held_so(PATH, SIZE, BACKWARD, decltype(lanes)::value, decltype(per)::value))
      if (h.lanes == lanes && h.per == per) {
        found = true;
        f(lanes, per);
      }
  };
  using std::integral_constant;
  lanes_per(integral_constant<int, 8>{}, integral_constant<int, 8>{});
  lanes_per(integral_constant<int, 16>{}, integral_constant<int, 8>{});
  lanes_per(integral_constant<int, 32>{}, integral_constant<int, 8>{});
  lanes_per(integral_constant<int, 32>{}, integral_constant<int, 16>{});
  lanes_per(integral_constant<int, 0>{}, integral_constant<int, 8>{});
  lanes_per(integral_constant<int, 0>{}, integral_constant<int, 16>{});
  if (!found) throw Error("sandwich norm: no kernel holds such a row");
}

int ring_per(long long width) { return width <= 4096 ? 8 : 16; }
RingPlan forward_ring(const so3lr_sandwich_norm_args &a, Path path) {
  if (path != kWide || !ring_takes(a.width, a.dtype == SO3LR_FLOAT32 ? 4 : 2, false)) return RingPlan{0, 0, 0};
  const int per = ring_per(a.width);
  return ring_plan(a.rows, row_threads(a.width, per), per == 8 ? 1024 : 512, 2,
                   (a.gate ? 3 : 2) * a.width * (a.dtype == SO3LR_FLOAT32 ? 4 : 2));
}
struct BackPlan {
  Path path;
  Hold hold;
  int grid, threads;
  RingPlan ring;
};
BackPlan back_plan(const so3lr_sandwich_norm_backward_args &a) {
  RowTensors t{a.dtype == SO3LR_FLOAT32 ? 4 : 2};
  t.add(a.dy, a.dy_stride);
  t.add(a.ds, a.ds_stride);
  t.add(a.s, a.s_stride);
  t.add(a.x, a.x_stride);
  if (a.residual_scale) t.add(a.residual, a.residual_stride);
  t.add(a.gate, a.gate_stride);
  t.add(a.dx, a.dx_stride);
  t.add(a.dresidual, a.dresidual_stride);
  t.add(a.dgate, a.dgate_stride);
  BackPlan p;
  p.path = t.path(a.width, aligned(a.weight, 0, 1, 16) && aligned(a.next_weight, 0, 1, 16) &&
                               aligned(a.residual_scale, 0, 1, 16));
  p.hold = sandwich_hold(a.width, p.path, t.size, true);
  p.ring = RingPlan{0, 0, 0};
  if (p.path == kWide && ring_takes(a.width, t.size, true)) {
    const int per = ring_per(a.width), threads = row_threads(a.width, per);
    const RingPlan r = ring_plan(a.rows, threads, 512, 2,
                                 (3 + (a.ds ? 1 : 0) + (a.gate ? 1 : 0) + (a.residual_scale ? 1 : 0)) * a.width * t.size);
    if (r.stages >= 2) {
      p.ring = r;
      p.grid = r.grid;
      p.threads = threads;
      return p;
    }
  }
  if (p.hold.per == 0) {
    p.threads = 512;
    p.grid = int(std::min<long long>(a.rows, kSmCount));
    return p;
  }
  p.threads = p.hold.lanes ? kTeamThreads : row_threads(a.width, p.hold.per);
  const int per_sm = p.hold.lanes ? 2 : std::max(1, 512 / p.threads);
  p.grid = int(std::min<long long>(team_grid(p.hold, a.rows).x, (long long)kSmCount * per_sm));
  if (p.path == kShifted && p.hold.lanes == 0) p.grid = (p.grid + 7) / 8 * 8;
  return p;
}

}  // namespace

void launch_sandwich_norm(const so3lr_sandwich_norm_args &a, cudaStream_t s) {
  by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    by_weight<T>(a.dtype, a.weight_dtype, [&](auto w) {
      using W = decltype(w);
      RowTensors t{int(sizeof(T))};
      t.add(a.x, a.x_stride);
      t.add(a.residual, a.residual_stride);
      t.add(a.gate, a.gate_stride);
      t.add(a.s, a.s_stride);
      t.add(a.y, a.y_stride);
      const Path chosen = t.path(a.width, aligned(a.weight, 0, 1, 16) && aligned(a.next_weight, 0, 1, 16) &&
                                              aligned(a.residual_scale, 0, 1, 16));
      const RingPlan r = forward_ring(a, chosen);
      if (r.stages >= 2 && a.rows > 2 * r.grid) {
        auto go = [&](auto kernel) {
          allow_dynamic_smem(reinterpret_cast<const void *>(kernel), 227 * 1024 - 1024);
          launch(kernel, r.grid, row_threads(a.width, ring_per(a.width)), r.smem, s, a, r.stages, wait_limit(),
                 1.0f / float(a.width), float(a.eps));
        };
        if constexpr (sizeof(T) == 2) {
          if (ring_per(a.width) == 8) {
            go(&k_sandwich_ring<T, W, 8>);
            return;
          }
        }
        go(&k_sandwich_ring<T, W, 16>);
        return;
      }
      by_path(chosen, [&](auto path) {
        constexpr Path PATH = decltype(path)::value;
        constexpr int VEC = chunk_of(PATH, sizeof(T));
        const Hold h = sandwich_hold(a.width, PATH, sizeof(T), false);
        by_sandwich_hold<PATH, sizeof(T), false>(h, [&](auto lanes, auto per) {
          constexpr int L = decltype(lanes)::value, N = decltype(per)::value / VEC;
          launch(k_sandwich<T, W, VEC, N, L, PATH == kShifted>, team_grid(h, a.rows), team_block(h, a.width), 0, s, a,
                 1.0f / float(a.width), float(a.eps));
        });
      });
    });
  });
}

long long sandwich_norm_backward_bytes(const so3lr_sandwich_norm_backward_args &a) {
  return (long long)back_plan(a).grid * 3 * a.width * 4;
}

void launch_sandwich_norm_backward(const so3lr_sandwich_norm_backward_args &a, void *workspace, cudaStream_t s) {
  by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    by_weight<T>(a.dtype, a.weight_dtype, [&](auto w) {
      using W = decltype(w);
      const BackPlan p = back_plan(a);
      float *partial = static_cast<float *>(workspace);
      const float inv = 1.0f / float(a.width), eps = float(a.eps);
      if (p.grid > 0 && p.ring.stages) {
        auto go = [&](auto kernel) {
          allow_dynamic_smem(reinterpret_cast<const void *>(kernel), 227 * 1024 - 1024);
          launch(kernel, p.grid, p.threads, p.ring.smem, s, a, partial, p.ring.stages, wait_limit(), inv, eps);
        };
        if (ring_per(a.width) == 8)
          go(&k_sandwich_backward_ring<T, W, 8>);
        else
          go(&k_sandwich_backward_ring<T, W, 16>);
      } else if (p.grid > 0 && p.hold.per == 0) {
        auto go = [&](auto kernel) {
          allow_dynamic_smem(reinterpret_cast<const void *>(kernel), 3 * 16384 * sizeof(float));
          launch(kernel, p.grid, p.threads, 3 * a.width * sizeof(float), s, a, partial, inv, eps);
        };
        if (p.path == kWide)
          go(&k_sandwich_backward_long<T, W, 16 / sizeof(T)>);
        else
          go(&k_sandwich_backward_long<T, W, 1>);
      } else if (p.grid > 0) {
        by_path(p.path, [&](auto path) {
          constexpr Path PATH = decltype(path)::value;
          constexpr int VEC = chunk_of(PATH, sizeof(T));
          by_sandwich_hold<PATH, sizeof(T), true>(p.hold, [&](auto lanes, auto per) {
            constexpr int L = decltype(lanes)::value, N = decltype(per)::value / VEC;
            launch(k_sandwich_backward<T, W, VEC, N, L, PATH == kShifted>, p.grid, p.threads,
                   L ? kTeamThreads / (L ? L : 1) * a.width * sizeof(float) : 0, s, a, partial, inv, eps);
          });
        });
      }
      const Sums<W> sums{{static_cast<W *>(a.dweight), static_cast<W *>(a.dnext_weight),
                          static_cast<W *>(a.dresidual_scale)}};
      launch(k_column_sums<W>, dim3(unsigned((a.width + 31) / 32), a.residual_scale ? 3 : 2), dim3(32, 32), 0, s,
             p.grid, int(a.width), partial, sums);
    });
  });
}

}  // namespace so3lr_b200
