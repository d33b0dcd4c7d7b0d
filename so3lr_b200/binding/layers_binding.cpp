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
#include <optional>
#include <sstream>
#include <stdexcept>
#include <string>
#include <utility>

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
                           METHOD(feed_forward_backward, 7), METHOD(status, 1), METHOD(set_wait_limit, 1), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_layers", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__layers() {
  PyObject *runtime = PyImport_ImportModule("so3lr_b200.runtime");
  if (!runtime) return nullptr;
  g_error = PyObject_GetAttrString(runtime, "So3lrError");
  Py_DECREF(runtime);
  return g_error ? PyModule_Create(&g_module) : nullptr;
}
