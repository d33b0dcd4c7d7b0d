// extern "C" boundary of the row-wise feed-forward layers: argument checks, then
// the launchers of rows.cu and dense.cu. Every refusal happens before a launch.
#include "layers.hpp"

#include <string>

#include "checks.hpp"

using so3lr_b200::Error;
using namespace so3lr_b200::checks;

namespace {

void check(const so3lr_rms_norm_args *a) {
  const char *call = "so3lr_rms_norm";
  require(a != nullptr, "so3lr_rms_norm: args is NULL");
  length(call, "rows", a->rows, 0, kMaxLength);
  length(call, "width", a->width, 1, 16384);
  type(call, "dtype", a->dtype);
  if (a->weight_dtype != a->dtype && a->weight_dtype != SO3LR_FLOAT32)
    throw Error("so3lr_rms_norm: weight_dtype must be dtype or SO3LR_FLOAT32");
  require(a->eps >= 0 && a->eps < 1e30, "so3lr_rms_norm: eps must be finite and not negative");
  require((a->y != nullptr) != (a->codes != nullptr) || a->rows == 0,
          "so3lr_rms_norm: exactly one of y and codes must be given");
  require((a->residual != nullptr) == (a->s != nullptr) || a->rows == 0,
          "so3lr_rms_norm: s must be given with a residual, and only then");
  const std::size_t e = bytes_of(a->dtype);
  matrix(call, "x", a->x, a->x_stride, a->rows, a->width, e, false);
  if (a->residual) {
    matrix(call, "residual", a->residual, a->residual_stride, a->rows, a->width, e, false);
    matrix(call, "s", a->s, a->s_stride, a->rows, a->width, e, true);
  }
  pointer(call, "weight", a->weight, bytes_of(a->weight_dtype));
  if (a->y) matrix(call, "y", a->y, a->y_stride, a->rows, a->width, e, true);
  if (a->codes) {
    matrix(call, "codes", a->codes, a->codes_stride, a->rows, a->width, 1, true);
    if (a->rows) pointer(call, "scales", a->scales, 4);
  }
}

void check_sizes(const so3lr_rms_norm_backward_args *a) {
  const char *call = "so3lr_rms_norm_backward";
  require(a != nullptr, "so3lr_rms_norm_backward: args is NULL");
  length(call, "rows", a->rows, 0, kMaxLength);
  length(call, "width", a->width, 1, 16384);
  type(call, "dtype", a->dtype);
  if (a->weight_dtype != a->dtype && a->weight_dtype != SO3LR_FLOAT32)
    throw Error("so3lr_rms_norm_backward: weight_dtype must be dtype or SO3LR_FLOAT32");
}
void check(const so3lr_rms_norm_backward_args *a) {
  const char *call = "so3lr_rms_norm_backward";
  check_sizes(a);
  require(a->eps >= 0 && a->eps < 1e30, "so3lr_rms_norm_backward: eps must be finite and not negative");
  const std::size_t e = bytes_of(a->dtype);
  matrix(call, "dy", a->dy, a->dy_stride, a->rows, a->width, e, false);
  matrix(call, "s", a->s, a->s_stride, a->rows, a->width, e, false);
  if (a->ds) matrix(call, "ds", a->ds, a->ds_stride, a->rows, a->width, e, false);
  matrix(call, "dx", a->dx, a->dx_stride, a->rows, a->width, e, true);
  pointer(call, "weight", a->weight, bytes_of(a->weight_dtype));
  pointer(call, "dweight", a->dweight, bytes_of(a->weight_dtype));
}

void check_sizes(const so3lr_int8_linear_args *a) {
  const char *call = "so3lr_int8_linear";
  require(a != nullptr, "so3lr_int8_linear: args is NULL");
  length(call, "rows", a->rows, 0, kMaxLength);
  length(call, "n", a->n, 1, kMaxLength);
  length(call, "k", a->k, 1, 131071);
  type(call, "out_dtype", a->out_dtype);
}
void check(const so3lr_int8_linear_args *a) {
  const char *call = "so3lr_int8_linear";
  check_sizes(a);
  matrix(call, "a", a->a, a->a_stride, a->rows, a->k, 1, false);
  matrix(call, "b", a->b, a->b_stride, a->n, a->k, 1, false);
  if (a->rows) pointer(call, "a_scales", a->a_scales, 4);
  pointer(call, "b_scales", a->b_scales, 4);
  if (a->bias) pointer(call, "bias", a->bias, 4);
  matrix(call, "y", a->y, a->y_stride, a->rows, a->n, bytes_of(a->out_dtype), true);
}

void check(const so3lr_gate_int8_args *a) {
  const char *call = "so3lr_gate_int8";
  require(a != nullptr, "so3lr_gate_int8: args is NULL");
  length(call, "rows", a->rows, 0, kMaxLength);
  length(call, "hidden", a->hidden, 1, 32768);
  type(call, "dtype", a->dtype);
  matrix(call, "gu", a->gu, a->gu_stride, a->rows, 2 * a->hidden, bytes_of(a->dtype), false);
  matrix(call, "codes", a->codes, a->codes_stride, a->rows, a->hidden, 1, true);
  if (a->rows) pointer(call, "scales", a->scales, 4);
}

void check(const so3lr_dequantize_int8_args *a) {
  const char *call = "so3lr_dequantize_int8";
  require(a != nullptr, "so3lr_dequantize_int8: args is NULL");
  length(call, "rows", a->rows, 0, kMaxLength);
  length(call, "width", a->width, 1, kMaxLength);
  type(call, "dtype", a->dtype);
  matrix(call, "codes", a->codes, a->codes_stride, a->rows, a->width, 1, false);
  if (a->rows) pointer(call, "scales", a->scales, 4);
  matrix(call, "out", a->out, a->out_stride, a->rows, a->width, bytes_of(a->dtype), true);
}

template <class A>
void check_feed_forward_sizes(const char *call, const A *a) {
  if (!a) throw Error(std::string(call) + ": args is NULL");
  length(call, "rows", a->rows, 0, kMaxLength);
  length(call, "width", a->width, 1, 1 << 20);
  length(call, "hidden", a->hidden, 1, 1 << 20);
  type(call, "dtype", a->dtype, true);
}
template <class A>
void check_feed_forward_inputs(const char *call, const A *a) {
  matrix(call, "x", a->x, a->x_stride, a->rows, a->width, 2, false);
  matrix(call, "w_gate", a->w_gate, a->w_gate_stride, a->hidden, a->width, 2, false);
  matrix(call, "w_up", a->w_up, a->w_up_stride, a->hidden, a->width, 2, false);
  matrix(call, "w_down", a->w_down, a->w_down_stride, a->width, a->hidden, 2, false);
}
void check(const so3lr_feed_forward_args *a) {
  const char *call = "so3lr_feed_forward";
  check_feed_forward_sizes(call, a);
  check_feed_forward_inputs(call, a);
  matrix(call, "y", a->y, a->y_stride, a->rows, a->width, 2, true);
  if (a->h) matrix(call, "h", a->h, a->hidden, a->rows, a->hidden, 2, true);
  if (a->gu) pointer(call, "gu", a->gu, 16);
}
void check(const so3lr_feed_forward_backward_args *a) {
  const char *call = "so3lr_feed_forward_backward";
  check_feed_forward_sizes(call, a);
  check_feed_forward_inputs(call, a);
  matrix(call, "dy", a->dy, a->dy_stride, a->rows, a->width, 2, false);
  matrix(call, "h", a->h, a->hidden, a->rows, a->hidden, 2, false);
  if (a->gu) pointer(call, "gu", a->gu, 16);
  matrix(call, "dx", a->dx, a->dx_stride, a->rows, a->width, 2, true);
  pointer(call, "dw_gate", a->dw_gate, 2);
  pointer(call, "dw_up", a->dw_up, 2);
  pointer(call, "dw_down", a->dw_down, 2);
}

}  // namespace

extern "C" {

int so3lr_layers_status(char *err, size_t errlen) {
  return guarded(err, errlen, [&] {
    if (const int where = so3lr_b200::take_gave_up()) throw Error(so3lr_b200::gave_up_message(where));
  });
}

void so3lr_layers_wait_limit(long long cycles) { so3lr_b200::set_wait_limit(cycles); }

int so3lr_rms_norm(const so3lr_rms_norm_args *args, void *stream, char *err, size_t errlen) {
  return guarded(err, errlen, [&] {
    check(args);
    if (args->rows == 0) return;
    so3lr_b200::check_gave_up();
    so3lr_b200::launch_rms_norm(*args, static_cast<cudaStream_t>(stream));
  });
}

long long so3lr_rms_norm_backward_workspace(const so3lr_rms_norm_backward_args *args) {
  return sized([&] {
    check_sizes(args);
    return so3lr_b200::rms_norm_backward_bytes(*args);
  });
}
int so3lr_rms_norm_backward(const so3lr_rms_norm_backward_args *args, void *workspace, long long workspace_bytes,
                            void *stream, char *err, size_t errlen) {
  return guarded(err, errlen, [&] {
    check(args);
    workspace_is("so3lr_rms_norm_backward", workspace, workspace_bytes, so3lr_b200::rms_norm_backward_bytes(*args));
    so3lr_b200::check_gave_up();
    so3lr_b200::launch_rms_norm_backward(*args, workspace, static_cast<cudaStream_t>(stream));
  });
}

long long so3lr_int8_linear_workspace(const so3lr_int8_linear_args *args) {
  return sized([&] {
    check_sizes(args);
    return so3lr_b200::int8_linear_bytes(*args);
  });
}
int so3lr_int8_linear(const so3lr_int8_linear_args *args, void *workspace, long long workspace_bytes, void *stream,
                      char *err, size_t errlen) {
  return guarded(err, errlen, [&] {
    check(args);
    workspace_is("so3lr_int8_linear", workspace, workspace_bytes, so3lr_b200::int8_linear_bytes(*args));
    if (args->rows == 0) return;
    so3lr_b200::check_gave_up();
    so3lr_b200::launch_int8_linear(*args, workspace, static_cast<cudaStream_t>(stream));
  });
}

int so3lr_gate_int8(const so3lr_gate_int8_args *args, void *stream, char *err, size_t errlen) {
  return guarded(err, errlen, [&] {
    check(args);
    if (args->rows == 0) return;
    so3lr_b200::check_gave_up();
    so3lr_b200::launch_gate_int8(*args, static_cast<cudaStream_t>(stream));
  });
}

int so3lr_dequantize_int8(const so3lr_dequantize_int8_args *args, void *stream, char *err, size_t errlen) {
  return guarded(err, errlen, [&] {
    check(args);
    if (args->rows == 0) return;
    so3lr_b200::check_gave_up();
    so3lr_b200::launch_dequantize_int8(*args, static_cast<cudaStream_t>(stream));
  });
}

long long so3lr_feed_forward_workspace(const so3lr_feed_forward_args *args) {
  return sized([&] {
    check_feed_forward_sizes("so3lr_feed_forward", args);
    return so3lr_b200::feed_forward_bytes(*args);
  });
}
long long so3lr_feed_forward_keep(const so3lr_feed_forward_args *args) {
  return sized([&] {
    check_feed_forward_sizes("so3lr_feed_forward", args);
    return so3lr_b200::feed_forward_keep(*args);
  });
}
int so3lr_feed_forward(const so3lr_feed_forward_args *args, void *workspace, long long workspace_bytes, void *stream,
                       char *err, size_t errlen) {
  return guarded(err, errlen, [&] {
    check(args);
    workspace_is("so3lr_feed_forward", workspace, workspace_bytes, so3lr_b200::feed_forward_bytes(*args));
    if (args->rows == 0) return;
    so3lr_b200::check_gave_up();
    so3lr_b200::launch_feed_forward(*args, workspace, static_cast<cudaStream_t>(stream));
  });
}

long long so3lr_feed_forward_backward_workspace(const so3lr_feed_forward_backward_args *args) {
  return sized([&] {
    check_feed_forward_sizes("so3lr_feed_forward_backward", args);
    return so3lr_b200::feed_forward_backward_bytes(*args);
  });
}
int so3lr_feed_forward_backward(const so3lr_feed_forward_backward_args *args, void *workspace,
                                long long workspace_bytes, void *stream, char *err, size_t errlen) {
  return guarded(err, errlen, [&] {
    check(args);
    workspace_is("so3lr_feed_forward_backward", workspace, workspace_bytes,
                 so3lr_b200::feed_forward_backward_bytes(*args));
    so3lr_b200::check_gave_up();
    so3lr_b200::launch_feed_forward_backward(*args, workspace, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
