// What a block is made of besides its feed-forward layer (include/so3lr_b200.h): the norms
// on both sides of its boundary and the dense layer. Launchers behind the C entry points of
// block.cpp. Arguments have been checked there.
#pragma once

#include "layers.hpp"

namespace so3lr_b200 {

// sandwich.cu
void launch_sandwich_norm(const so3lr_sandwich_norm_args &a, cudaStream_t s);
long long sandwich_norm_backward_bytes(const so3lr_sandwich_norm_backward_args &a);
void launch_sandwich_norm_backward(const so3lr_sandwich_norm_backward_args &a, void *workspace, cudaStream_t s);

// dense.cu
long long linear_bytes(const so3lr_linear_args &a);
void launch_linear(const so3lr_linear_args &a, void *workspace, cudaStream_t s);
long long linear_backward_bytes(const so3lr_linear_backward_args &a);
void launch_linear_backward(const so3lr_linear_backward_args &a, void *workspace, cudaStream_t s);

// linear.cu: dz (where dz is not dy itself) and, with `partial`, the bias gradient
long long linear_elementwise_bytes(const so3lr_linear_backward_args &a);
void launch_linear_elementwise(const so3lr_linear_backward_args &a, void *dz, long long dz_stride, float *partial,
                               cudaStream_t s);

// few_rows.cu. Few rows are those where the weights times the groups of 16 rows are below a limit
// that grows with the contraction, as for the other products. Measured even (us in this kernel
// and the tcgen05 one): 64 to 8192 channels 56 rows (6.2, 5.6), 256 to 4096 64 (5.6, 6.2), 1024 to
// 1024 128 (8.9, 10.0), 1024 to 4096 32 (9.0, 9.7), 2048 to 2048 32 (8.2, 8.4), 4096 to 1024 48 (7.6,
// 8.8), 4096 to 4096 16 (13.4, 15.3).
inline bool few_rows(const so3lr_linear_args &a) {
  return few_rows(a.rows, 2 * a.n * a.k, a.k < 1408 ? 2 + a.k / 64 : 24);
}
void launch_linear_few(const so3lr_linear_args &a, cudaStream_t s);

}  // namespace so3lr_b200
