// Python module so3lr_b200._layers: the row-wise feed-forward layers' C entry points
// (include/so3lr_b200.h) on torch tensors. Argument checks, output and workspace
// allocation (torch's allocator) and the current stream; no arithmetic. A call of a
// single row costs a few microseconds of kernel time, so this path is compiled: the
// same steps through ctypes took 16 us for rms_norm_int8, most of it Python and
// torch.empty.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/TracerMode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdio>
#include <deque>
#include <optional>
#include <sstream>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "so3lr_b200.h"

namespace {

using at::Tensor;

PyObject *g_error = nullptr;  // so3lr_b200.runtime.So3lrError

struct Refusal : std::runtime_error {  // becomes a ValueError
  using std::runtime_error::runtime_error;
};
template <class... A>
[[noreturn]] void refuse(const A &...parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw Refusal(s.str());
}

const char *name_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kChar: return "torch.int8";
    case at::kByte: return "torch.uint8";
    case at::kLong: return "torch.int64";
    default: return c10::toString(t);
  }
}
int float_type(at::ScalarType t, const char *what, bool half_only = false) {
  if (t == at::kBFloat16) return SO3LR_BFLOAT16;
  if (t == at::kHalf) return SO3LR_FLOAT16;
  if (t == at::kFloat && !half_only) return SO3LR_FLOAT32;
  refuse(what, half_only ? " must be one of torch.bfloat16, torch.float16, got "
                         : " must be one of torch.float32, torch.bfloat16, torch.float16, got ",
         name_of(t));
}

const Tensor &tensor(PyObject *o, const char *what) {
  if (!THPVariable_Check(o)) refuse(what, " must be a tensor");
  const Tensor &t = THPVariable_Unpack(o);
  // the results would be without a tangent of their own, and what is computed from them wrong
  if (t._fw_grad(0).defined()) refuse(what, " has a forward-mode tangent, which these calls do not carry on");
  return t;
}

double number(PyObject *o, const char *what) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(what, " must be a number");
  }
  return v;
}

// A matrix of rows: all leading dimensions of a tensor, with one row stride
struct Rows {
  void *data;
  int64_t rows, width, stride;
  at::ScalarType type;
  c10::Device device;
};
Rows rows_of(const Tensor &t, const char *what) {
  if (t.dim() < 1) refuse(what, " must have at least one dimension");
  if (!t.is_cuda()) refuse(what, " must be on a CUDA device, got ", t.device().str(), " (there is no CPU path)");
  const auto size = t.sizes(), stride = t.strides();
  const int64_t d = t.dim(), width = size[d - 1];
  if (width < 1) refuse(what, " must have rows of at least one element");
  if (width > 1 && stride[d - 1] != 1) refuse(what, " must have a contiguous last dimension");
  int64_t rows = 1, step = width;
  bool first = true;
  for (int64_t i = d - 2; i >= 0; --i) {
    if (size[i] != 1 && t.numel() > 0) {
      if (first)
        step = stride[i];
      else if (stride[i] != step * rows)
        refuse("the leading dimensions of ", what, " cannot be seen as rows of one stride");
      first = false;
    }
    rows *= size[i];
  }
  return Rows{t.data_ptr(), rows, width, step, t.scalar_type(), t.device()};
}
Rows rows_like(const Tensor &t, const char *what, const Rows &like, at::ScalarType type, int64_t rows, int64_t width) {
  const Rows r = rows_of(t, what);
  if (r.device != like.device) refuse(what, " is on ", r.device.str(), ", the other tensors are on ", like.device.str());
  if (r.type != type) refuse(what, " must be ", name_of(type), ", got ", name_of(r.type));
  if (width >= 0 && r.width != width) refuse(what, " must have rows of ", width, " elements, got ", r.width);
  if (rows >= 0 && r.rows != rows) refuse(what, " must have ", rows, " rows, got ", r.rows);
  return r;
}
void *vector_of(const Tensor &t, const char *what, const Rows &like, int64_t length, at::ScalarType type,
                std::optional<at::ScalarType> or_type = std::nullopt) {
  if (t.dim() != 1 || t.size(0) != length || t.device() != like.device)
    refuse(what, " must be a 1-D tensor of ", length, " elements on ", like.device.str());
  if (t.scalar_type() != type && t.scalar_type() != or_type)
    refuse(what, " must be ", name_of(type), or_type ? " or " : "", or_type ? name_of(*or_type) : "", ", got ",
           name_of(t.scalar_type()));
  if (length > 1 && t.stride(0) != 1) refuse(what, " must be contiguous");
  return t.data_ptr();
}

Tensor empty(at::IntArrayRef size, at::ScalarType type, c10::Device device) {
  return at::detail::empty_cuda(size, type, device, std::nullopt);
}
// 8-bit rows that start on 16-byte boundaries, as int8_linear reads them without a copy
Tensor empty_codes(int64_t rows, int64_t width, c10::Device device) {
  const int64_t padded = (width + 15) / 16 * 16;
  Tensor t = empty({rows, padded}, at::kChar, device);
  return padded == width ? t : t.narrow(1, 0, width);
}
// `like`'s leading dimensions, last dimension `width`
at::DimVector shaped(const Tensor &like, int64_t width) {
  at::DimVector s(like.sizes().begin(), like.sizes().end());
  s.back() = width;
  return s;
}

void check(int rc, const char *err) {
  if (rc) throw std::runtime_error(err);
}
void *stream_of(c10::Device d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }

// The C call with a workspace of the size that it asks for
template <class A, class Size, class Call>
void with_workspace(const A &a, c10::Device device, Size size, Call call) {
  char err[1024] = "";
  const long long need = size(&a);
  Tensor ws;
  if (need > 0) ws = empty({int64_t(need)}, at::kByte, device);
  check(call(&a, need > 0 ? ws.data_ptr() : nullptr, need > 0 ? need : 0, stream_of(device), err, sizeof err), err);
}

PyObject *wrap(Tensor t) { return THPVariable_Wrap(std::move(t)); }
PyObject *none() { Py_RETURN_NONE; }
template <class... O>
PyObject *tuple(O... o) {
  PyObject *t = PyTuple_New(sizeof...(o));
  Py_ssize_t i = 0;
  (PyTuple_SET_ITEM(t, i++, o), ...);
  return t;
}

using Args = PyObject *const *;

// rms_norm(x, weight, residual, eps, quantize) -> (y | codes, scales | None, s)
PyObject *rms_norm(Args o) {
  const Tensor &x = tensor(o[0], "x"), &w = tensor(o[1], "weight");
  const bool quantize = PyObject_IsTrue(o[4]);
  const Rows r = rows_of(x, "x");
  const c10::cuda::CUDAGuard guard(r.device);
  so3lr_rms_norm_args a{};
  a.rows = r.rows;
  a.width = r.width;
  a.dtype = float_type(r.type, "x");
  a.eps = number(o[3], "eps");
  a.x = r.data;
  a.x_stride = r.stride;
  a.weight = vector_of(w, "weight", r, r.width, r.type, at::kFloat);
  a.weight_dtype = w.scalar_type() == at::kFloat ? SO3LR_FLOAT32 : a.dtype;
  Tensor s;
  if (o[2] != Py_None) {
    const Tensor &res = tensor(o[2], "residual");
    if (res.sizes() != x.sizes()) refuse("residual must have the shape of x, got ", res.sizes(), " and ", x.sizes());
    const Rows q = rows_like(res, "residual", r, r.type, r.rows, r.width);
    s = empty(x.sizes(), r.type, r.device);
    a.residual = q.data;
    a.residual_stride = q.stride;
    a.s = s.data_ptr();
    a.s_stride = r.width;
  }
  Tensor y, scales;
  if (quantize) {
    y = empty_codes(r.rows, r.width, r.device);
    scales = empty({r.rows}, at::kFloat, r.device);
    a.codes = static_cast<signed char *>(y.data_ptr());
    a.codes_stride = y.stride(0);
    a.scales = static_cast<float *>(scales.data_ptr());
  } else {
    y = empty(x.sizes(), r.type, r.device);
    a.y = y.data_ptr();
    a.y_stride = r.width;
  }
  char err[1024] = "";
  check(so3lr_rms_norm(&a, stream_of(r.device), err, sizeof err), err);
  PyObject *stream = o[0];
  if (s.defined())
    stream = wrap(s);
  else
    Py_INCREF(stream);
  return tuple(wrap(y), quantize ? wrap(scales) : none(), stream);
}

// rms_norm_backward(dy, s, weight, ds, eps) -> (dx, dweight)
PyObject *rms_norm_backward(Args o) {
  const Tensor &dy = tensor(o[0], "dy"), &s = tensor(o[1], "s"), &w = tensor(o[2], "weight");
  const Rows r = rows_of(s, "s");
  const c10::cuda::CUDAGuard guard(r.device);
  so3lr_rms_norm_backward_args a{};
  a.rows = r.rows;
  a.width = r.width;
  a.dtype = float_type(r.type, "s");
  a.eps = number(o[4], "eps");
  a.s = r.data;
  a.s_stride = r.stride;
  a.weight = vector_of(w, "weight", r, r.width, r.type, at::kFloat);
  a.weight_dtype = w.scalar_type() == at::kFloat ? SO3LR_FLOAT32 : a.dtype;
  const Rows d = rows_like(dy, "dy", r, r.type, r.rows, r.width);
  a.dy = d.data;
  a.dy_stride = d.stride;
  if (o[3] != Py_None) {
    const Rows e = rows_like(tensor(o[3], "ds"), "ds", r, r.type, r.rows, r.width);
    a.ds = e.data;
    a.ds_stride = e.stride;
  }
  Tensor dx = empty(s.sizes(), r.type, r.device), dw = empty({r.width}, w.scalar_type(), r.device);
  a.dx = dx.data_ptr();
  a.dx_stride = r.width;
  a.dweight = dw.data_ptr();
  with_workspace(a, r.device, so3lr_rms_norm_backward_workspace, so3lr_rms_norm_backward);
  return tuple(wrap(dx), wrap(dw));
}

at::ScalarType dtype_of(PyObject *o, const char *what) {
  if (!THPDtype_Check(o)) refuse(what, " must be a torch.dtype");
  return reinterpret_cast<THPDtype *>(o)->scalar_type;
}

// int8_linear(a, a_scales, b, b_scales, bias, out_dtype) -> y
PyObject *int8_linear(Args o) {
  const Tensor &x = tensor(o[0], "a"), &w = tensor(o[2], "b");
  const Rows r = rows_of(x, "a");
  if (r.type != at::kChar) refuse("a must be torch.int8, got ", name_of(r.type));
  const c10::cuda::CUDAGuard guard(r.device);
  const Rows b = rows_like(w, "b", r, at::kChar, -1, r.width);
  if (b.rows < 1) refuse("b must have at least one row");
  const at::ScalarType out = dtype_of(o[5], "out_dtype");
  so3lr_int8_linear_args a{};
  a.rows = r.rows;
  a.n = b.rows;
  a.k = r.width;
  a.out_dtype = float_type(out, "out_dtype");
  a.a = static_cast<const signed char *>(r.data);
  a.a_stride = r.stride;
  a.a_scales = static_cast<const float *>(vector_of(tensor(o[1], "a_scales"), "a_scales", r, r.rows, at::kFloat));
  a.b = static_cast<const signed char *>(b.data);
  a.b_stride = b.stride;
  a.b_scales = static_cast<const float *>(vector_of(tensor(o[3], "b_scales"), "b_scales", r, b.rows, at::kFloat));
  if (o[4] != Py_None)
    a.bias = static_cast<const float *>(vector_of(tensor(o[4], "bias"), "bias", r, b.rows, at::kFloat));
  Tensor y = empty(shaped(x, b.rows), out, r.device);
  a.y = y.data_ptr();
  a.y_stride = b.rows;
  with_workspace(a, r.device, so3lr_int8_linear_workspace, so3lr_int8_linear);
  return wrap(y);
}

// gate_int8(gu) -> (codes, scales)
PyObject *gate_int8(Args o) {
  const Rows r = rows_of(tensor(o[0], "gu"), "gu");
  const int type = float_type(r.type, "gu");
  if (r.width % 2) refuse("gu must hold g and u side by side: an even width, got ", r.width);
  const c10::cuda::CUDAGuard guard(r.device);
  Tensor codes = empty_codes(r.rows, r.width / 2, r.device), scales = empty({r.rows}, at::kFloat, r.device);
  so3lr_gate_int8_args a{};
  a.rows = r.rows;
  a.hidden = r.width / 2;
  a.dtype = type;
  a.gu = r.data;
  a.gu_stride = r.stride;
  a.codes = static_cast<signed char *>(codes.data_ptr());
  a.codes_stride = codes.stride(0);
  a.scales = static_cast<float *>(scales.data_ptr());
  char err[1024] = "";
  check(so3lr_gate_int8(&a, stream_of(r.device), err, sizeof err), err);
  return tuple(wrap(codes), wrap(scales));
}

// dequantize_int8(codes, scales, dtype) -> values
PyObject *dequantize_int8(Args o) {
  const Tensor &codes = tensor(o[0], "codes");
  const Rows r = rows_of(codes, "codes");
  if (r.type != at::kChar) refuse("codes must be torch.int8, got ", name_of(r.type));
  const c10::cuda::CUDAGuard guard(r.device);
  const at::ScalarType out = dtype_of(o[2], "dtype");
  so3lr_dequantize_int8_args a{};
  a.rows = r.rows;
  a.width = r.width;
  a.dtype = float_type(out, "dtype");
  a.codes = static_cast<const signed char *>(r.data);
  a.codes_stride = r.stride;
  a.scales = static_cast<const float *>(vector_of(tensor(o[1], "scales"), "scales", r, r.rows, at::kFloat));
  Tensor y = empty(codes.sizes(), out, r.device);
  a.out = y.data_ptr();
  a.out_stride = r.width;
  char err[1024] = "";
  check(so3lr_dequantize_int8(&a, stream_of(r.device), err, sizeof err), err);
  return wrap(y);
}

// x, w_gate, w_up, w_down of either feed-forward call
template <class A>
Rows feed_forward_operands(A &a, Args o) {
  const Rows x = rows_of(tensor(o[0], "x"), "x");
  a.dtype = float_type(x.type, "x", true);
  const Rows g = rows_like(tensor(o[1], "w_gate"), "w_gate", x, x.type, -1, x.width);
  if (g.rows < 1) refuse("w_gate must have at least one row");
  const Rows u = rows_like(tensor(o[2], "w_up"), "w_up", x, x.type, g.rows, x.width);
  const Rows d = rows_like(tensor(o[3], "w_down"), "w_down", x, x.type, x.width, g.rows);
  a.rows = x.rows;
  a.width = x.width;
  a.hidden = g.rows;
  a.x = x.data;
  a.x_stride = x.stride;
  a.w_gate = g.data;
  a.w_gate_stride = g.stride;
  a.w_up = u.data;
  a.w_up_stride = u.stride;
  a.w_down = d.data;
  a.w_down_stride = d.stride;
  return x;
}

// feed_forward(x, w_gate, w_up, w_down, keep) -> y, or with keep (y, h, gu | None)
PyObject *feed_forward(Args o) {
  so3lr_feed_forward_args a{};
  const Rows r = feed_forward_operands(a, o);
  const bool keep = PyObject_IsTrue(o[4]);
  const c10::cuda::CUDAGuard guard(r.device);
  Tensor y = empty(tensor(o[0], "x").sizes(), r.type, r.device), h, gu;
  a.y = y.data_ptr();
  a.y_stride = r.width;
  if (keep) {
    h = empty({r.rows, int64_t(a.hidden)}, r.type, r.device);
    a.h = h.data_ptr();
    const long long bytes = so3lr_feed_forward_keep(&a);
    if (bytes > 0) {
      gu = empty({int64_t(bytes / 4)}, at::kFloat, r.device);
      a.gu = static_cast<float *>(gu.data_ptr());
    }
  }
  with_workspace(a, r.device, so3lr_feed_forward_workspace, so3lr_feed_forward);
  if (!keep) return wrap(y);
  return tuple(wrap(y), wrap(h), gu.defined() ? wrap(gu) : none());
}

// feed_forward_backward(x, w_gate, w_up, w_down, dy, h, gu) -> (dx, dw_gate, dw_up, dw_down)
PyObject *feed_forward_backward(Args o) {
  so3lr_feed_forward_backward_args a{};
  const Rows r = feed_forward_operands(a, o);
  const int64_t hidden = a.hidden;
  const c10::cuda::CUDAGuard guard(r.device);
  const Rows d = rows_like(tensor(o[4], "dy"), "dy", r, r.type, r.rows, r.width);
  a.dy = d.data;
  a.dy_stride = d.stride;
  const Tensor &h = tensor(o[5], "saved");
  const char *wrong = "saved does not come from feed_forward_train on these tensors";
  if (h.dim() != 2 || h.size(0) != r.rows || h.size(1) != hidden || h.scalar_type() != r.type ||
      h.device() != r.device || !h.is_contiguous())
    refuse(wrong);
  a.h = h.data_ptr();
  if (o[6] != Py_None) {
    const Tensor &gu = tensor(o[6], "saved");
    if (gu.scalar_type() != at::kFloat || gu.device() != r.device || !gu.is_contiguous() ||
        gu.numel() != (r.rows + 31) / 32 * 32 * hidden * 2)
      refuse(wrong);
    a.gu = static_cast<const float *>(gu.data_ptr());
  }
  Tensor dx = empty(tensor(o[0], "x").sizes(), r.type, r.device), dwg = empty({hidden, r.width}, r.type, r.device),
         dwu = empty({hidden, r.width}, r.type, r.device), dwd = empty({r.width, hidden}, r.type, r.device);
  a.dx = dx.data_ptr();
  a.dx_stride = r.width;
  a.dw_gate = dwg.data_ptr();
  a.dw_up = dwu.data_ptr();
  a.dw_down = dwd.data_ptr();
  with_workspace(a, r.device, so3lr_feed_forward_backward_workspace, so3lr_feed_forward_backward);
  return tuple(wrap(dx), wrap(dwg), wrap(dwu), wrap(dwd));
}

// a whole number of a Python int
int whole(PyObject *o, const char *what) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(what, " must be a whole number");
  }
  return int(v);
}

// linear(x, weight, bias | None, residual | None, activation, keep) -> y, or with keep (y, z | None)
PyObject *linear(Args o) {
  const Tensor &x = tensor(o[0], "x");
  const Rows r = rows_of(x, "x");
  so3lr_linear_args a{};
  a.dtype = a.bias_dtype = float_type(r.type, "x", true);
  const Rows w = rows_like(tensor(o[1], "weight"), "weight", r, r.type, -1, r.width);
  if (w.rows < 1) refuse("weight must have at least one row");
  const bool keep = PyObject_IsTrue(o[5]);
  const c10::cuda::CUDAGuard guard(r.device);
  a.rows = r.rows;
  a.n = w.rows;
  a.k = r.width;
  a.activation = whole(o[4], "activation");
  a.x = r.data;
  a.x_stride = r.stride;
  a.w = w.data;
  a.w_stride = w.stride;
  if (o[2] != Py_None) {
    const Tensor &bias = tensor(o[2], "bias");
    a.bias = vector_of(bias, "bias", r, w.rows, r.type, at::kFloat);
    if (bias.scalar_type() == at::kFloat) a.bias_dtype = SO3LR_FLOAT32;
  }
  const at::DimVector shape = shaped(x, w.rows);
  if (o[3] != Py_None) {
    const Tensor &residual = tensor(o[3], "residual");
    if (residual.sizes() != at::IntArrayRef(shape))
      refuse("residual must have the shape of the result, ", at::IntArrayRef(shape), ", got ", residual.sizes());
    const Rows q = rows_like(residual, "residual", r, r.type, r.rows, w.rows);
    a.residual = q.data;
    a.residual_stride = q.stride;
  }
  Tensor y = empty(shape, r.type, r.device), z;
  a.y = y.data_ptr();
  a.y_stride = w.rows;
  if (keep && a.activation != SO3LR_NO_ACTIVATION) {  // rows on 16-byte boundaries
    const int64_t padded = (w.rows + 7) / 8 * 8;
    z = empty({r.rows, padded}, r.type, r.device);
    a.z = z.data_ptr();
    a.z_stride = padded;
    if (padded != w.rows) z = z.narrow(1, 0, w.rows);
  }
  with_workspace(a, r.device, so3lr_linear_workspace, so3lr_linear);
  if (!keep) return wrap(y);
  return tuple(wrap(y), z.defined() ? wrap(z) : none());
}

// linear_backward(dy, x, weight, z | None, activation, bias dtype | None, dx wanted, dweight wanted)
// -> (dx | None, dweight | None, dbias | None)
PyObject *linear_backward(Args o) {
  const Tensor &x = tensor(o[1], "x");
  const Rows r = rows_of(x, "x");
  so3lr_linear_backward_args a{};
  a.dtype = a.bias_dtype = float_type(r.type, "x", true);
  const Rows w = rows_like(tensor(o[2], "weight"), "weight", r, r.type, -1, r.width);
  if (w.rows < 1) refuse("weight must have at least one row");
  const c10::cuda::CUDAGuard guard(r.device);
  const Rows d = rows_like(tensor(o[0], "dy"), "dy", r, r.type, r.rows, w.rows);
  a.rows = r.rows;
  a.n = w.rows;
  a.k = r.width;
  a.activation = whole(o[4], "activation");
  a.dy = d.data;
  a.dy_stride = d.stride;
  a.x = r.data;
  a.x_stride = r.stride;
  a.w = w.data;
  a.w_stride = w.stride;
  if (a.activation != SO3LR_NO_ACTIVATION) {
    if (o[3] == Py_None) refuse("saved does not come from linear_train on these tensors");
    const Rows z = rows_like(tensor(o[3], "saved"), "saved", r, r.type, r.rows, w.rows);
    a.z = z.data;
    a.z_stride = z.stride;
  }
  Tensor dx, dw, dbias;
  if (PyObject_IsTrue(o[6])) {
    dx = empty(x.sizes(), r.type, r.device);
    a.dx = dx.data_ptr();
    a.dx_stride = r.width;
  }
  if (PyObject_IsTrue(o[7])) {
    dw = empty({w.rows, r.width}, r.type, r.device);
    a.dw = dw.data_ptr();
  }
  if (o[5] != Py_None) {
    const at::ScalarType t = dtype_of(o[5], "bias");
    if (t != r.type && t != at::kFloat) refuse("bias must be ", name_of(r.type), " or torch.float32, got ", name_of(t));
    if (t == at::kFloat) a.bias_dtype = SO3LR_FLOAT32;
    dbias = empty({w.rows}, t, r.device);
    a.dbias = dbias.data_ptr();
  }
  with_workspace(a, r.device, so3lr_linear_backward_workspace, so3lr_linear_backward);
  return tuple(dx.defined() ? wrap(dx) : none(), dw.defined() ? wrap(dw) : none(),
               dbias.defined() ? wrap(dbias) : none());
}

// x, residual, weight, next_weight, gate | None, residual_scale | None of either sandwich call
template <class A>
Rows sandwich_operands(A &a, Args o, PyObject *eps) {
  const Tensor &x = tensor(o[0], "x"), &residual = tensor(o[1], "residual"), &w = tensor(o[2], "weight");
  const Rows r = rows_of(x, "x");
  a.rows = r.rows;
  a.width = r.width;
  a.dtype = float_type(r.type, "x");
  a.eps = number(eps, "eps");
  a.x = r.data;
  a.x_stride = r.stride;
  if (residual.sizes() != x.sizes())
    refuse("residual must have the shape of x, got ", residual.sizes(), " and ", x.sizes());
  const Rows q = rows_like(residual, "residual", r, r.type, r.rows, r.width);
  a.residual = q.data;
  a.residual_stride = q.stride;
  a.weight = vector_of(w, "weight", r, r.width, r.type, at::kFloat);
  a.weight_dtype = w.scalar_type() == at::kFloat ? SO3LR_FLOAT32 : a.dtype;
  a.next_weight = vector_of(tensor(o[3], "next_weight"), "next_weight", r, r.width, w.scalar_type());
  if (o[4] != Py_None) {
    const Tensor &gate = tensor(o[4], "gate");
    if (gate.sizes() != x.sizes()) refuse("gate must have the shape of x, got ", gate.sizes(), " and ", x.sizes());
    const Rows g = rows_like(gate, "gate", r, r.type, r.rows, r.width);
    a.gate = g.data;
    a.gate_stride = g.stride;
  }
  if (o[5] != Py_None)
    a.residual_scale = vector_of(tensor(o[5], "residual_scale"), "residual_scale", r, r.width, w.scalar_type());
  return r;
}

// sandwich_norm(x, residual, weight, next_weight, gate | None, residual_scale | None, eps) -> (y, s)
PyObject *sandwich_norm(Args o) {
  so3lr_sandwich_norm_args a{};
  const Rows r = sandwich_operands(a, o, o[6]);
  const c10::cuda::CUDAGuard guard(r.device);
  const Tensor &x = tensor(o[0], "x");
  Tensor y = empty(x.sizes(), r.type, r.device), s = empty(x.sizes(), r.type, r.device);
  a.y = y.data_ptr();
  a.s = s.data_ptr();
  a.y_stride = a.s_stride = r.width;
  char err[1024] = "";
  check(so3lr_sandwich_norm(&a, stream_of(r.device), err, sizeof err), err);
  return tuple(wrap(y), wrap(s));
}

// sandwich_norm_backward(x, residual, weight, next_weight, gate | None, residual_scale | None, dy, ds | None, s, eps)
// -> (dx, dresidual, dweight, dnext_weight, dgate | None, dresidual_scale | None)
PyObject *sandwich_norm_backward(Args o) {
  so3lr_sandwich_norm_backward_args a{};
  const Rows r = sandwich_operands(a, o, o[9]);
  const c10::cuda::CUDAGuard guard(r.device);
  const Tensor &x = tensor(o[0], "x"), &w = tensor(o[2], "weight");
  const Rows d = rows_like(tensor(o[6], "dy"), "dy", r, r.type, r.rows, r.width);
  a.dy = d.data;
  a.dy_stride = d.stride;
  if (o[7] != Py_None) {
    const Rows e = rows_like(tensor(o[7], "ds"), "ds", r, r.type, r.rows, r.width);
    a.ds = e.data;
    a.ds_stride = e.stride;
  }
  const Rows s = rows_like(tensor(o[8], "s"), "s", r, r.type, r.rows, r.width);
  a.s = s.data;
  a.s_stride = s.stride;
  Tensor dx = empty(x.sizes(), r.type, r.device), dresidual = empty(x.sizes(), r.type, r.device), dgate, dscale,
         dw = empty({r.width}, w.scalar_type(), r.device), dnext = empty({r.width}, w.scalar_type(), r.device);
  a.dx = dx.data_ptr();
  a.dresidual = dresidual.data_ptr();
  a.dx_stride = a.dresidual_stride = r.width;
  a.dweight = dw.data_ptr();
  a.dnext_weight = dnext.data_ptr();
  if (o[4] != Py_None) {
    dgate = empty(x.sizes(), r.type, r.device);
    a.dgate = dgate.data_ptr();
    a.dgate_stride = r.width;
  }
  if (a.residual_scale) {
    dscale = empty({r.width}, w.scalar_type(), r.device);
    a.dresidual_scale = dscale.data_ptr();
  }
  with_workspace(a, r.device, so3lr_sandwich_norm_backward_workspace, so3lr_sandwich_norm_backward);
  return tuple(wrap(dx), wrap(dresidual), wrap(dw), wrap(dnext), dgate.defined() ? wrap(dgate) : none(),
               dscale.defined() ? wrap(dscale) : none());
}

// A list of tensors (or of None) as borrowed references; the list object must outlive it
struct List {
  PyObject *fast;
  List(PyObject *o, const char *what) : fast(PySequence_Fast(o, "")) {
    if (!fast) {
      PyErr_Clear();
      refuse(what, " must be a list of tensors");
    }
  }
  ~List() { Py_DECREF(fast); }
  List(const List &) = delete;
  Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(fast); }
  PyObject *operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(fast, i); }
};
// one tensor of a list, contiguous, with `n` elements of one of two types
const Tensor &element(const List &list, Py_ssize_t i, const char *what, c10::Device device, int64_t n,
                      at::ScalarType type, std::optional<at::ScalarType> or_type = std::nullopt) {
  const Tensor &t = tensor(list[i], what);
  if (t.layout() != at::kStrided) refuse(what, "[", i, "] must be a dense tensor");
  if (t.device() != device) refuse(what, "[", i, "] is on ", t.device().str(), ", the other tensors are on ", device.str());
  if (t.scalar_type() != type && t.scalar_type() != or_type)
    refuse(what, "[", i, "] must be ", name_of(type), or_type ? " or " : "", or_type ? name_of(*or_type) : "", ", got ",
           name_of(t.scalar_type()));
  if (t.numel() != n) refuse(what, "[", i, "] must have ", n, " elements, got ", t.numel());
  if (!t.is_contiguous()) refuse(what, "[", i, "] must be contiguous");
  return t;
}

constexpr int64_t kScaleBlock = 256;

// One AdamW call: its arguments as the library takes them. The Python objects must outlive it.
struct AdamwCall {
  List params;
  so3lr_adamw_args a{};
  std::vector<so3lr_adamw_tensor> tensors;
  c10::Device device{c10::kCUDA};
  explicit AdamwCall(Args o);
  AdamwCall(const AdamwCall &) = delete;
  void check_arguments() const {
    char err[1024] = "";
    check(so3lr_adamw_check(&a, err, sizeof err), err);
  }
  void run() const;
};
// params, grads, exp_avgs, exp_avg_sqs, steps, exp_avg_scales | None, exp_avg_sq_scales | None, masters | None, lr,
// beta1, beta2, eps, weight_decay
AdamwCall::AdamwCall(Args o) : params(o[0], "params") {
  const List grads(o[1], "grads"), ms(o[2], "exp_avgs"), vs(o[3], "exp_avg_sqs");
  const Py_ssize_t count = params.size();
  std::optional<List> m_scales, v_scales, masters, counters;
  if (o[5] != Py_None) m_scales.emplace(o[5], "exp_avg_scales");
  if (o[6] != Py_None) v_scales.emplace(o[6], "exp_avg_sq_scales");
  if (o[7] != Py_None) masters.emplace(o[7], "masters");
  if (!THPVariable_Check(o[4])) counters.emplace(o[4], "steps");
  auto same = [&](const List &l, const char *what) {
    if (l.size() != count) refuse(what, " must have as many tensors as params, ", count, ", got ", l.size());
  };
  same(grads, "grads");
  same(ms, "exp_avgs");
  same(vs, "exp_avg_sqs");
  if (m_scales) same(*m_scales, "exp_avg_scales");
  if (v_scales) same(*v_scales, "exp_avg_sq_scales");
  if (masters) same(*masters, "masters");
  if (counters) same(*counters, "steps");
  a.beta1 = number(o[9], "betas");
  a.beta2 = number(o[10], "betas");
  a.eps = number(o[11], "eps");
  a.weight_decay = number(o[12], "weight_decay");
  a.count = count;
  if (count == 0) return;
  const Tensor &first = tensor(params[0], "params");
  device = first.device();
  if (!first.is_cuda()) refuse("params must be on a CUDA device, got ", device.str(), " (there is no CPU path)");
  if (THPVariable_Check(o[8])) {
    const Tensor &lr = tensor(o[8], "lr");
    if (lr.device() != device || lr.scalar_type() != at::kFloat || lr.numel() != 1)
      refuse("lr must be a number or a torch.float32 tensor of one element on ", device.str());
    a.lr_device = static_cast<const float *>(lr.data_ptr());
  } else {
    a.lr = number(o[8], "lr");
  }
  long long *steps = nullptr;
  if (!counters) {
    const Tensor &t = tensor(o[4], "steps");
    if (t.dim() != 1 || t.size(0) != count || t.device() != device || t.scalar_type() != at::kLong || !t.is_contiguous())
      refuse("steps must be a contiguous 1-D torch.int64 tensor of ", count, " elements on ", device.str(),
             ", or a list of tensors of one");
    steps = reinterpret_cast<long long *>(t.data_ptr());
  }
  tensors.resize(count);
  for (Py_ssize_t i = 0; i < count; ++i) {
    so3lr_adamw_tensor &e = tensors[i];
    const Tensor &p = tensor(params[i], "params");
    e.n = p.numel();
    const at::ScalarType t = p.scalar_type();
    e.dtype = float_type(t, "params");
    e.param = element(params, i, "params", device, e.n, t).data_ptr();
    const Tensor &g = element(grads, i, "grads", device, e.n, t, at::kFloat);
    e.grad = g.data_ptr();
    e.grad_dtype = g.scalar_type() == at::kFloat ? SO3LR_FLOAT32 : e.dtype;
    const bool eight = m_scales && (*m_scales)[i] != Py_None;
    if (eight != (v_scales && (*v_scales)[i] != Py_None))
      refuse("exp_avg_scales[", i, "] and exp_avg_sq_scales[", i, "] must be given together");
    e.exp_avg = element(ms, i, "exp_avgs", device, e.n, eight ? at::kChar : at::kFloat).data_ptr();
    e.exp_avg_sq = element(vs, i, "exp_avg_sqs", device, e.n, eight ? at::kByte : at::kFloat).data_ptr();
    if (eight) {
      const int64_t blocks = (e.n + kScaleBlock - 1) / kScaleBlock;
      e.exp_avg_scale = static_cast<float *>(element(*m_scales, i, "exp_avg_scales", device, blocks, at::kFloat).data_ptr());
      e.exp_avg_sq_scale =
          static_cast<float *>(element(*v_scales, i, "exp_avg_sq_scales", device, blocks, at::kFloat).data_ptr());
    }
    if (masters && (*masters)[i] != Py_None)
      e.master = static_cast<float *>(element(*masters, i, "masters", device, e.n, at::kFloat).data_ptr());
    e.step = counters ? reinterpret_cast<long long *>(element(*counters, i, "steps", device, 1, at::kLong).data_ptr())
                      : steps + i;
  }
  a.tensors = tensors.data();
}
void AdamwCall::run() const {
  if (a.count == 0) return;
  const c10::cuda::CUDAGuard guard(device);
  with_workspace(a, device, so3lr_adamw_workspace, so3lr_adamw);
  // what autograd has kept of the parameters for a backward pass to come is no longer what it was
  for (Py_ssize_t i = 0; i < a.count; ++i)
    if (const Tensor &p = THPVariable_Unpack(params[i]); !p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
}

// adamw_step(an AdamwCall's arguments) -> None
PyObject *adamw_step(Args o) {
  AdamwCall(o).run();
  return none();
}

// adamw_steps(a list of tuples of such arguments) -> None: nothing is launched before the last call's arguments
// have been checked
PyObject *adamw_steps(Args o) {
  const List list(o[0], "calls");
  std::deque<AdamwCall> calls;
  for (Py_ssize_t i = 0; i < list.size(); ++i) {
    if (!PyTuple_Check(list[i]) || PyTuple_GET_SIZE(list[i]) != 13) refuse("calls must be tuples of 13 arguments");
    calls.emplace_back(&PyTuple_GET_ITEM(list[i], 0));
  }
  if (calls.size() > 1)
    for (const AdamwCall &c : calls) c.check_arguments();
  for (const AdamwCall &c : calls) c.run();
  return none();
}

// uniform(a list of tensors) -> whether the dense ones are contiguous and all are on one device
PyObject *uniform(Args o) {
  const List list(o[0], "tensors");
  for (Py_ssize_t i = 0; i < list.size(); ++i) {
    const Tensor &t = tensor(list[i], "tensors");
    if (t.layout() == at::kStrided && !t.is_contiguous()) Py_RETURN_FALSE;
    if (t.device() != tensor(list[0], "tensors").device()) Py_RETURN_FALSE;
  }
  Py_RETURN_TRUE;
}

// moment_values(codes, scales, dtype) -> values
PyObject *moment_values(Args o) {
  const Tensor &codes = tensor(o[0], "codes"), &scales = tensor(o[1], "scales");
  if (!codes.is_cuda()) refuse("codes must be on a CUDA device, got ", codes.device().str(), " (there is no CPU path)");
  if (codes.scalar_type() != at::kChar && codes.scalar_type() != at::kByte)
    refuse("codes must be torch.int8 or torch.uint8, got ", name_of(codes.scalar_type()));
  if (!codes.is_contiguous()) refuse("codes must be contiguous");
  const int64_t blocks = (codes.numel() + kScaleBlock - 1) / kScaleBlock;
  if (scales.device() != codes.device() || scales.scalar_type() != at::kFloat || scales.numel() != blocks ||
      !scales.is_contiguous())
    refuse("scales must be a contiguous torch.float32 tensor of ", blocks, " elements on ", codes.device().str());
  const c10::cuda::CUDAGuard guard(codes.device());
  const at::ScalarType out = dtype_of(o[2], "dtype");
  so3lr_moment_values_args a{};
  a.n = codes.numel();
  a.is_signed = codes.scalar_type() == at::kChar;
  a.dtype = float_type(out, "dtype");
  a.codes = codes.data_ptr();
  a.scales = static_cast<const float *>(scales.data_ptr());
  Tensor y = empty(codes.sizes(), out, codes.device());
  a.values = y.data_ptr();
  char err[1024] = "";
  check(so3lr_moment_values(&a, stream_of(codes.device()), err, sizeof err), err);
  return wrap(y);
}

// status(device index) -> None
PyObject *status(Args o) {
  const c10::cuda::CUDAGuard guard(c10::Device(c10::kCUDA, c10::DeviceIndex(PyLong_AsLong(o[0]))));
  char err[1024] = "";
  check(so3lr_layers_status(err, sizeof err), err);
  return none();
}

// set_wait_limit(cycles) -> None
PyObject *set_wait_limit(Args o) {
  so3lr_layers_wait_limit(PyLong_AsLongLong(o[0]));
  return none();
}

// No C++ exception leaves the module: refusals become ValueError, failures of the
// library So3lrError, torch's own errors RuntimeError.
template <PyObject *(*F)(Args), int N>
PyObject *method(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  try {
    // it would record the results as constants
    if (at::tracer::impl::is_dispatch_enabled()) refuse("torch.jit.trace cannot record the feed-forward layers");
    PyObject *r = F(args);
    if (PyErr_Occurred()) {
      Py_XDECREF(r);
      return nullptr;
    }
    return r;
  } catch (const Refusal &e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::Error &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception &e) {
    PyErr_SetString(g_error, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown exception");
  }
  return nullptr;
}

#define METHOD(f, n) \
  { #f, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&method<f, n>)), METH_FASTCALL, nullptr }
PyMethodDef g_methods[] = {METHOD(rms_norm, 5),        METHOD(rms_norm_backward, 5), METHOD(int8_linear, 6),
                           METHOD(gate_int8, 1),       METHOD(dequantize_int8, 3),   METHOD(feed_forward, 5),
                           METHOD(feed_forward_backward, 7), METHOD(linear, 6),          METHOD(linear_backward, 8),
                           METHOD(sandwich_norm, 7),
                           METHOD(sandwich_norm_backward, 10), METHOD(adamw_step, 13),   METHOD(adamw_steps, 1),
                           METHOD(uniform, 1),
                           METHOD(moment_values, 3),   METHOD(status, 1), METHOD(set_wait_limit, 1), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_layers", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__layers() {
  PyObject *runtime = PyImport_ImportModule("so3lr_b200.runtime");
  if (!runtime) return nullptr;
  g_error = PyObject_GetAttrString(runtime, "So3lrError");
  Py_DECREF(runtime);
  return g_error ? PyModule_Create(&g_module) : nullptr;
}
