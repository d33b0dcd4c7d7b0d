// Products of the feed-forward layers: simple kernels, one thread per output
// element from 16 x 16 shared-memory tiles, operands through strided views.
#include "layers_common.cuh"

namespace so3lr_b200 {
namespace {

constexpr int kTile = 16;

template <class T>
__device__ __forceinline__ auto at(const View &v, long long r, long long c) {
  return static_cast<const T *>(v.data)[r * v.row + c * v.col];
}

// one element of A (m x k) times B (n x k), transposed; all threads of the block call it
template <class T, class Acc>
__device__ Acc product(const View &A, const View &B, long long m, long long n, long long k, long long row,
                       long long col) {
  __shared__ Acc ta[kTile][kTile + 1], tb[kTile][kTile + 1];
  Acc sum = 0;
  const long long brow = col - threadIdx.x + threadIdx.y;
  for (long long k0 = 0; k0 < k; k0 += kTile) {
    const long long c = k0 + threadIdx.x;
    ta[threadIdx.y][threadIdx.x] = row < m && c < k ? Acc(at<T>(A, row, c)) : Acc(0);
    tb[threadIdx.y][threadIdx.x] = brow < n && c < k ? Acc(at<T>(B, brow, c)) : Acc(0);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTile; ++i) sum += ta[threadIdx.y][i] * tb[threadIdx.x][i];
    __syncthreads();
  }
  return sum;
}

__device__ __forceinline__ long long tile_row() { return (long long)blockIdx.x * kTile + threadIdx.y; }
__device__ __forceinline__ long long tile_col() { return (long long)blockIdx.y * kTile + threadIdx.x; }
dim3 grid_of(long long m, long long n) {
  return dim3(unsigned((m + kTile - 1) / kTile), unsigned((n + kTile - 1) / kTile));
}

template <class O>
__global__ void k_int8_linear(const so3lr_int8_linear_args a) {
  const long long r = tile_row(), c = tile_col();
  const int sum = product<signed char, int>(View{a.a, a.a_stride, 1}, View{a.b, a.b_stride, 1}, a.rows, a.n, a.k, r, c);
  if (r >= a.rows || c >= a.n) return;
  float y = float(sum) * a.a_scales[r] * a.b_scales[c];
  if (a.bias) y += a.bias[c];
  static_cast<O *>(a.y)[r * a.y_stride + c] = from_float<O>(y);
}

// C = A1 B1^T (+ A2 B2^T)
template <class T>
__global__ void k_product(View A1, View B1, View A2, View B2, long long m, long long n, long long k, T *C,
                          long long c_stride) {
  const long long r = tile_row(), c = tile_col();
  float v = product<T, float>(A1, B1, m, n, k, r, c);
  if (A2.data) v += product<T, float>(A2, B2, m, n, k, r, c);
  if (r < m && c < n) C[r * c_stride + c] = from_float<T>(v);
}

template <class T>
__global__ void k_gated(View X, View G, View U, long long m, long long n, long long k, T *H) {
  const long long r = tile_row(), c = tile_col();
  const float g = product<T, float>(X, G, m, n, k, r, c), u = product<T, float>(X, U, m, n, k, r, c);
  if (r < m && c < n) H[r * n + c] = from_float<T>(silu_f32(g) * u);
}

template <class T>
__global__ void k_gated_backward(View X, View G, View U, View DY, View DT, long long m, long long n, long long k,
                                 T *H, T *DG, T *DU) {
  const long long r = tile_row(), c = tile_col();
  const float g = product<T, float>(X, G, m, n, k, r, c), u = product<T, float>(X, U, m, n, k, r, c);
  const float dh = product<T, float>(DY, DT, m, n, k, r, c);
  if (r >= m || c >= n) return;
  const float sg = __fdividef(1.0f, 1.0f + __expf(-g));
  H[r * n + c] = from_float<T>(g * sg * u);
  DU[r * n + c] = from_float<T>(dh * g * sg);
  DG[r * n + c] = from_float<T>(dh * u * sg * (1.0f + g * (1.0f - sg)));
}

template <class F>
void by_half(int dtype, F &&f) {
  if (dtype == SO3LR_BFLOAT16)
    f(__nv_bfloat16{});
  else
    f(__half{});
}
const dim3 kBlock(kTile, kTile);

template <class T>
void multiply(View A, View B, View A2, View B2, long long m, long long n, long long k, void *c, long long c_stride,
              cudaStream_t s) {
  k_product<T><<<grid_of(m, n), kBlock, 0, s>>>(A, B, A2, B2, m, n, k, static_cast<T *>(c), c_stride);
  SO3_LAUNCH("product");
}

}  // namespace

long long int8_linear_bytes(const so3lr_int8_linear_args &) { return 0; }
void launch_int8_linear(const so3lr_int8_linear_args &a, void *, cudaStream_t s) {
  const dim3 grid = grid_of(a.rows, a.n);
  if (a.out_dtype == SO3LR_FLOAT32)
    k_int8_linear<float><<<grid, kBlock, 0, s>>>(a);
  else if (a.out_dtype == SO3LR_BFLOAT16)
    k_int8_linear<__nv_bfloat16><<<grid, kBlock, 0, s>>>(a);
  else
    k_int8_linear<__half><<<grid, kBlock, 0, s>>>(a);
  SO3_LAUNCH("int8_linear");
}

long long feed_forward_bytes(const so3lr_feed_forward_args &a) { return a.rows * a.hidden * 2; }
void launch_feed_forward(const so3lr_feed_forward_args &a, void *workspace, cudaStream_t s) {
  by_half(a.dtype, [&](auto t) {
    using T = decltype(t);
    k_gated<T><<<grid_of(a.rows, a.hidden), kBlock, 0, s>>>(
        View{a.x, a.x_stride, 1}, View{a.w_gate, a.w_gate_stride, 1}, View{a.w_up, a.w_up_stride, 1}, a.rows,
        a.hidden, a.width, static_cast<T *>(workspace));
    SO3_LAUNCH("gated");
    multiply<T>(View{workspace, a.hidden, 1}, View{a.w_down, a.w_down_stride, 1}, View{}, View{}, a.rows, a.width,
                a.hidden, a.y, a.y_stride, s);
  });
}

long long feed_forward_backward_bytes(const so3lr_feed_forward_backward_args &a) {
  return 3 * a.rows * a.hidden * 2;
}
void launch_feed_forward_backward(const so3lr_feed_forward_backward_args &a, void *workspace, cudaStream_t s) {
  by_half(a.dtype, [&](auto t) {
    using T = decltype(t);
    const long long R = a.rows, D = a.width, H = a.hidden;
    T *h = static_cast<T *>(workspace), *dg = h + R * H, *du = dg + R * H;
    if (R > 0) {
      k_gated_backward<T><<<grid_of(R, H), kBlock, 0, s>>>(
          View{a.x, a.x_stride, 1}, View{a.w_gate, a.w_gate_stride, 1}, View{a.w_up, a.w_up_stride, 1},
          View{a.dy, a.dy_stride, 1}, View{a.w_down, 1, a.w_down_stride}, R, H, D, h, dg, du);
      SO3_LAUNCH("gated_backward");
      multiply<T>(View{dg, H, 1}, View{a.w_gate, 1, a.w_gate_stride}, View{du, H, 1}, View{a.w_up, 1, a.w_up_stride},
                  R, D, H, a.dx, a.dx_stride, s);
    }
    multiply<T>(View{dg, 1, H}, View{a.x, 1, a.x_stride}, View{}, View{}, H, D, R, a.dw_gate, D, s);
    multiply<T>(View{du, 1, H}, View{a.x, 1, a.x_stride}, View{}, View{}, H, D, R, a.dw_up, D, s);
    multiply<T>(View{a.dy, 1, a.dy_stride}, View{h, 1, H}, View{}, View{}, D, H, R, a.dw_down, H, s);
  });
}

}  // namespace so3lr_b200
