// extern "C" boundary of the norms on both sides of a block and of the dense layer:
// argument checks, then the launchers of sandwich.cu and dense.cu. Every refusal happens before a launch.
#include "block.hpp"

#include "checks.hpp"

using so3lr_b200::Error;
using namespace so3lr_b200::checks;

namespace {

template <class A>
void check_norm_sizes(const char *call, const A *a) {
  if (!a) throw Error(std::string(call) + ": args is NULL");
  length(call, "rows", a->rows, 0, kMaxLength);
  length(call, "width", a->width, 1, 16384);
  type(call, "dtype", a->dtype);
  if (a->weight_dtype != a->dtype && a->weight_dtype != SO3LR_FLOAT32)
    throw Error(name(call, "weight_dtype", "must be dtype or SO3LR_FLOAT32"));
}
template <class A>
void check_norm_inputs(const char *call, const A *a) {
  if (!(a->eps >= 0 && a->eps < 1e30)) throw Error(name(call, "eps", "must be finite and not negative"));
  const std::size_t e = bytes_of(a->dtype), we = bytes_of(a->weight_dtype);
  matrix(call, "x", a->x, a->x_stride, a->rows, a->width, e, false);
  if (a->gate) matrix(call, "gate", a->gate, a->gate_stride, a->rows, a->width, e, false);
  pointer(call, "weight", a->weight, we);
  pointer(call, "next_weight", a->next_weight, we);
  if (a->residual_scale) pointer(call, "residual_scale", a->residual_scale, we);
}
void check(const so3lr_sandwich_norm_args *a) {
  const char *call = "so3lr_sandwich_norm";
  check_norm_sizes(call, a);
  check_norm_inputs(call, a);
  const std::size_t e = bytes_of(a->dtype);
  matrix(call, "residual", a->residual, a->residual_stride, a->rows, a->width, e, false);
  matrix(call, "s", a->s, a->s_stride, a->rows, a->width, e, true);
  matrix(call, "y", a->y, a->y_stride, a->rows, a->width, e, true);
}
void check(const so3lr_sandwich_norm_backward_args *a) {
  const char *call = "so3lr_sandwich_norm_backward";
  check_norm_sizes(call, a);
  check_norm_inputs(call, a);
  const std::size_t e = bytes_of(a->dtype), we = bytes_of(a->weight_dtype);
  if (a->residual_scale) matrix(call, "residual", a->residual, a->residual_stride, a->rows, a->width, e, false);
  matrix(call, "dy", a->dy, a->dy_stride, a->rows, a->width, e, false);
  if (a->ds) matrix(call, "ds", a->ds, a->ds_stride, a->rows, a->width, e, false);
  matrix(call, "s", a->s, a->s_stride, a->rows, a->width, e, false);
  matrix(call, "dx", a->dx, a->dx_stride, a->rows, a->width, e, true);
  matrix(call, "dresidual", a->dresidual, a->dresidual_stride, a->rows, a->width, e, true);
  require((a->gate != nullptr) == (a->dgate != nullptr) || a->rows == 0,
          "so3lr_sandwich_norm_backward: dgate must be given with a gate, and only then");
  if (a->dgate) matrix(call, "dgate", a->dgate, a->dgate_stride, a->rows, a->width, e, true);
  pointer(call, "dweight", a->dweight, we);
  pointer(call, "dnext_weight", a->dnext_weight, we);
  require((a->residual_scale != nullptr) == (a->dresidual_scale != nullptr),
          "so3lr_sandwich_norm_backward: dresidual_scale must be given with a residual_scale, and only then");
  if (a->dresidual_scale) pointer(call, "dresidual_scale", a->dresidual_scale, we);
}

template <class A>
void check_linear_sizes(const char *call, const A *a) {
  if (!a) throw Error(std::string(call) + ": args is NULL");
  length(call, "rows", a->rows, 0, kMaxLength);
  length(call, "n", a->n, 1, 1 << 20);
  length(call, "k", a->k, 1, 1 << 20);
  type(call, "dtype", a->dtype, true);
  if (a->bias_dtype != a->dtype && a->bias_dtype != SO3LR_FLOAT32)
    throw Error(name(call, "bias_dtype", "must be dtype or SO3LR_FLOAT32"));
  if (a->activation < SO3LR_NO_ACTIVATION || a->activation > SO3LR_RELU)
    throw Error(name(call, "activation", "must be one of the five SO3LR_ activations"));
}
void check(const so3lr_linear_args *a) {
  const char *call = "so3lr_linear";
  check_linear_sizes(call, a);
  matrix(call, "x", a->x, a->x_stride, a->rows, a->k, 2, false);
  matrix(call, "w", a->w, a->w_stride, a->n, a->k, 2, false);
  if (a->bias) pointer(call, "bias", a->bias, bytes_of(a->bias_dtype));
  if (a->residual) matrix(call, "residual", a->residual, a->residual_stride, a->rows, a->n, 2, false);
  matrix(call, "y", a->y, a->y_stride, a->rows, a->n, 2, true);
  if (a->z) matrix(call, "z", a->z, a->z_stride, a->rows, a->n, 2, true);
}
void check(const so3lr_linear_backward_args *a) {
  const char *call = "so3lr_linear_backward";
  check_linear_sizes(call, a);
  matrix(call, "dy", a->dy, a->dy_stride, a->rows, a->n, 2, false);
  if (a->activation != SO3LR_NO_ACTIVATION) matrix(call, "z", a->z, a->z_stride, a->rows, a->n, 2, false);
  if (a->dx) {
    matrix(call, "w", a->w, a->w_stride, a->n, a->k, 2, false);
    matrix(call, "dx", a->dx, a->dx_stride, a->rows, a->k, 2, true);
  }
  if (a->dw) {
    matrix(call, "x", a->x, a->x_stride, a->rows, a->k, 2, false);
    pointer(call, "dw", a->dw, 2);
  }
  if (a->dbias) pointer(call, "dbias", a->dbias, bytes_of(a->bias_dtype));
}

}  // namespace

extern "C" {

long long so3lr_linear_workspace(const so3lr_linear_args *args) {
  return sized([&] {
    check_linear_sizes("so3lr_linear", args);
    return so3lr_b200::linear_bytes(*args);
  });
}
int so3lr_linear(const so3lr_linear_args *args, void *workspace, long long workspace_bytes, void *stream, char *err,
                 size_t errlen) {
  return guarded(err, errlen, [&] {
    check(args);
    workspace_is("so3lr_linear", workspace, workspace_bytes, so3lr_b200::linear_bytes(*args));
    if (args->rows == 0) return;
    so3lr_b200::check_gave_up();
    so3lr_b200::launch_linear(*args, workspace, static_cast<cudaStream_t>(stream));
  });
}

long long so3lr_linear_backward_workspace(const so3lr_linear_backward_args *args) {
  return sized([&] {
    check_linear_sizes("so3lr_linear_backward", args);
    return so3lr_b200::linear_backward_bytes(*args);
  });
}
int so3lr_linear_backward(const so3lr_linear_backward_args *args, void *workspace, long long workspace_bytes,
                          void *stream, char *err, size_t errlen) {
  return guarded(err, errlen, [&] {
    check(args);
    workspace_is("so3lr_linear_backward", workspace, workspace_bytes, so3lr_b200::linear_backward_bytes(*args));
    so3lr_b200::check_gave_up();
    so3lr_b200::launch_linear_backward(*args, workspace, static_cast<cudaStream_t>(stream));
  });
}

int so3lr_sandwich_norm(const so3lr_sandwich_norm_args *args, void *stream, char *err, size_t errlen) {
  return guarded(err, errlen, [&] {
    check(args);
    if (args->rows == 0) return;
    so3lr_b200::check_gave_up();
    so3lr_b200::launch_sandwich_norm(*args, static_cast<cudaStream_t>(stream));
  });
}

long long so3lr_sandwich_norm_backward_workspace(const so3lr_sandwich_norm_backward_args *args) {
  return sized([&] {
    check_norm_sizes("so3lr_sandwich_norm_backward", args);
    return so3lr_b200::sandwich_norm_backward_bytes(*args);
  });
}
int so3lr_sandwich_norm_backward(const so3lr_sandwich_norm_backward_args *args, void *workspace,
                                 long long workspace_bytes, void *stream, char *err, size_t errlen) {
  return guarded(err, errlen, [&] {
    check(args);
    workspace_is("so3lr_sandwich_norm_backward", workspace, workspace_bytes,
                 so3lr_b200::sandwich_norm_backward_bytes(*args));
    so3lr_b200::check_gave_up();
    so3lr_b200::launch_sandwich_norm_backward(*args, workspace, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
