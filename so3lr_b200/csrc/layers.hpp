// Row-wise feed-forward layers (include/so3lr_b200.h, "Row-wise feed-forward
// layers"): launchers behind the C entry points of layers.cpp. Arguments have
// been checked there.
#pragma once

#include <cstddef>

#include "../../include/so3lr_b200.h"
#include "common.cuh"

namespace so3lr_b200 {


// rows.cu
void launch_rms_norm(const so3lr_rms_norm_args &a, cudaStream_t s);
long long rms_norm_backward_bytes(const so3lr_rms_norm_backward_args &a);
void launch_rms_norm_backward(const so3lr_rms_norm_backward_args &a, void *workspace, cudaStream_t s);
void launch_gate_int8(const so3lr_gate_int8_args &a, cudaStream_t s);
void launch_dequantize_int8(const so3lr_dequantize_int8_args &a, cudaStream_t s);

// dense.cu
// Where a kernel whose bounded wait gave up says so, and the refusal of further calls after that.
int *gave_up_flag();
void check_gave_up();
long long int8_linear_bytes(const so3lr_int8_linear_args &a);
void launch_int8_linear(const so3lr_int8_linear_args &a, void *workspace, cudaStream_t s);
long long feed_forward_keep(const so3lr_feed_forward_args &a);
long long feed_forward_bytes(const so3lr_feed_forward_args &a);
void launch_feed_forward(const so3lr_feed_forward_args &a, void *workspace, cudaStream_t s);
long long feed_forward_backward_bytes(const so3lr_feed_forward_backward_args &a);
void launch_feed_forward_backward(const so3lr_feed_forward_backward_args &a, void *workspace, cudaStream_t s);

// few_rows.cu: the forward products for few rows, any alignment, no workspace but the
// hidden layer's. Its blocks read the weights once for every 16 rows, the tcgen05
// tiles (dense.cu) once for 256 but with about 3 us more of set-up a launch. Measured
// even: 64 rows of a 1.5 MB 8-bit weight (4.5 and 6.1 us; 96 rows 8.2 and 6.3), 128 rows
// through a block of 6.3 MB (14.6 and 16.1 us), 32 through one of 25 MB (17 and 21).
constexpr long long kFewRows = 16, kFewRowsMost = 256;
inline bool few_rows(long long rows, long long weight_bytes, long long limit) {
  return rows <= kFewRows || (rows <= kFewRowsMost && (rows + 15) / 16 * weight_bytes <= limit);
}
inline bool few_rows(const so3lr_int8_linear_args &a) { return few_rows(a.rows, a.n * a.k, 8 << 20); }
inline bool few_rows(const so3lr_feed_forward_args &a) {
  return !a.gu && few_rows(a.rows, 6 * a.width * a.hidden, 48 << 20);
}
void launch_int8_linear_few(const so3lr_int8_linear_args &a, cudaStream_t s);
void launch_feed_forward_few(const so3lr_feed_forward_args &a, void *h, long long h_stride, void *h_rest,
                             cudaStream_t s);

}  // namespace so3lr_b200
