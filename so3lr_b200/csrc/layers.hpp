// Row-wise feed-forward layers (include/so3lr_b200.h, "Row-wise feed-forward
// layers"): launchers behind the C entry points of layers.cpp. Arguments have
// been checked there.
#pragma once

#include <cstddef>
#include <string>

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
// Where a kernel whose bounded wait gave up on the current device says so (which wait, 0: none), the
// refusal of further calls after that, and reading and clearing it.
int *gave_up_flag();
void check_gave_up();
int take_gave_up();
std::string gave_up_message(int where);
// How long a kernel's wait may take, and where it says that it gave up; the limit of kernels queued from now on.
struct WaitLimit {
  int *err;
  long long cycles;
};
WaitLimit wait_limit();
void set_wait_limit(long long cycles);
long long int8_linear_bytes(const so3lr_int8_linear_args &a);
void launch_int8_linear(const so3lr_int8_linear_args &a, void *workspace, cudaStream_t s);
long long feed_forward_keep(const so3lr_feed_forward_args &a);
long long feed_forward_bytes(const so3lr_feed_forward_args &a);
void launch_feed_forward(const so3lr_feed_forward_args &a, void *workspace, cudaStream_t s);
long long feed_forward_backward_bytes(const so3lr_feed_forward_backward_args &a);
void launch_feed_forward_backward(const so3lr_feed_forward_backward_args &a, void *workspace, cudaStream_t s);

// few_rows.cu: the forward products for few rows, any alignment, no workspace but the
// hidden layer's. Its blocks read the weights once for every 16 rows, about 4 MB a
// microsecond; the tcgen05 tiles (dense.cu) read them once for 256, but a launch takes 3
// us or more, and longer the longer its contraction. Few rows are those where 16 or
// fewer, or the weights times the groups of 16 below a limit that grows with the
// contraction. Measured even (us in this kernel and that): 8-bit products of 64 to 8192
// channels 64 rows (5.3, 5.0), 1024 to 4096 48 (6.2, 6.0), 4096 to 1024 80 (7.9, 7.7);
// blocks of 64 x 8192 64 rows (13.0, 12.6), 256 x 4096 64 (13.0, 12.8), 1024 x 1024 96
// (15.3, 15.9), 2048 x 2048 32 (19.2, 21.6).
constexpr long long kFewRows = 16, kFewRowsMost = 256;
inline bool few_rows(long long rows, long long weight_bytes, long long limit_mb) {
  return rows <= kFewRows || (rows <= kFewRowsMost && (rows + 15) / 16 * weight_bytes <= limit_mb << 20);
}
inline bool few_rows(const so3lr_int8_linear_args &a) { return few_rows(a.rows, a.n * a.k, 2 + a.k / 200); }
inline bool few_rows(const so3lr_feed_forward_args &a) {
  return !a.gu && few_rows(a.rows, 6 * a.width * a.hidden, 12 + a.width / 40);
}
void launch_int8_linear_few(const so3lr_int8_linear_args &a, cudaStream_t s);
void launch_feed_forward_few(const so3lr_feed_forward_args &a, void *h, long long h_stride, void *h_rest,
                             cudaStream_t s);

}  // namespace so3lr_b200
