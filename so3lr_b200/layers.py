"""Row-wise feed-forward layers in low precision, on torch CUDA tensors.

The row-wise half of a transformer block over per-atom (or per-token) features:

* ``rms_norm`` (with the residual's addition), ``rms_norm_int8`` and the gradient
  ``rms_norm_backward``;
* ``int8_linear``, a product of 8-bit integers with a scale for each row of the
  activations and for each output channel, and ``gate_int8``, which stands
  between two of them in a feed-forward block; ``quantize_weight`` lays a weight
  out once, ``dequantize_int8`` reads 8-bit rows back;
* ``feed_forward``, the gated block y = (silu(x Wg^T) * (x Wu^T)) Wd^T, with
  ``feed_forward_train`` and ``feed_forward_backward`` for training.

``rms_norm`` and ``feed_forward`` record themselves for autograd when an argument
requires a gradient. ``FeedForwardBlock`` and ``Int8FeedForwardBlock`` run them
together: the pre-norm sublayer as it is trained, and the same weights served
in 8 bits.

The calls are the entry points of include/so3lr_b200.h ("Row-wise feed-forward
layers"): they queue kernels on the current torch stream of the tensors' GPU and
return; outputs and scratch come from torch's allocator. Rows are all leading
dimensions; the last dimension must be contiguous, rows may have any stride.
There is no CPU path: a tensor that is not on a GPU is refused.
"""
from __future__ import annotations

import ctypes as C
import threading

import torch

from .runtime import So3lrError, load_library

__all__ = ["rms_norm", "rms_norm_int8", "rms_norm_backward", "int8_linear", "gate_int8", "dequantize_int8",
           "quantize_weight", "feed_forward", "feed_forward_train", "feed_forward_backward", "FeedForwardBlock",
           "Int8FeedForwardBlock"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_HALF = {torch.bfloat16: 1, torch.float16: 2}
_ll, _p, _i, _d = C.c_longlong, C.c_void_p, C.c_int, C.c_double


class _RmsNorm(C.Structure):
    _fields_ = [("rows", _ll), ("width", _ll), ("dtype", _i), ("weight_dtype", _i), ("eps", _d), ("x", _p),
                ("x_stride", _ll), ("residual", _p), ("residual_stride", _ll), ("weight", _p), ("s", _p),
                ("s_stride", _ll), ("y", _p), ("y_stride", _ll), ("codes", _p), ("codes_stride", _ll),
                ("scales", _p)]


class _RmsNormBackward(C.Structure):
    _fields_ = [("rows", _ll), ("width", _ll), ("dtype", _i), ("weight_dtype", _i), ("eps", _d), ("dy", _p),
                ("dy_stride", _ll), ("s", _p), ("s_stride", _ll), ("weight", _p), ("ds", _p), ("ds_stride", _ll),
                ("dx", _p), ("dx_stride", _ll), ("dweight", _p)]


class _Int8Linear(C.Structure):
    _fields_ = [("rows", _ll), ("n", _ll), ("k", _ll), ("out_dtype", _i), ("a", _p), ("a_stride", _ll),
                ("a_scales", _p), ("b", _p), ("b_stride", _ll), ("b_scales", _p), ("bias", _p), ("y", _p),
                ("y_stride", _ll)]


class _GateInt8(C.Structure):
    _fields_ = [("rows", _ll), ("hidden", _ll), ("dtype", _i), ("gu", _p), ("gu_stride", _ll), ("codes", _p),
                ("codes_stride", _ll), ("scales", _p)]


class _DequantizeInt8(C.Structure):
    _fields_ = [("rows", _ll), ("width", _ll), ("dtype", _i), ("codes", _p), ("codes_stride", _ll), ("scales", _p),
                ("out", _p), ("out_stride", _ll)]


class _FeedForward(C.Structure):
    _fields_ = [("rows", _ll), ("width", _ll), ("hidden", _ll), ("dtype", _i), ("x", _p), ("x_stride", _ll),
                ("w_gate", _p), ("w_gate_stride", _ll), ("w_up", _p), ("w_up_stride", _ll), ("w_down", _p),
                ("w_down_stride", _ll), ("y", _p), ("y_stride", _ll), ("h", _p)]


class _FeedForwardBackward(C.Structure):
    _fields_ = [("rows", _ll), ("width", _ll), ("hidden", _ll), ("dtype", _i), ("dy", _p), ("dy_stride", _ll),
                ("x", _p), ("x_stride", _ll), ("w_gate", _p), ("w_gate_stride", _ll), ("w_up", _p),
                ("w_up_stride", _ll), ("w_down", _p), ("w_down_stride", _ll), ("h", _p), ("dx", _p), ("dx_stride", _ll),
                ("dw_gate", _p), ("dw_up", _p), ("dw_down", _p)]


_ERR_BYTES = 1024
_LOCAL = threading.local()  # a message buffer for each thread
_CALLS: dict = {}


def _lib():
    lib = load_library()
    if not _CALLS:
        plain = {"so3lr_rms_norm": _RmsNorm, "so3lr_gate_int8": _GateInt8, "so3lr_dequantize_int8": _DequantizeInt8}
        scratch = {"so3lr_rms_norm_backward": _RmsNormBackward, "so3lr_int8_linear": _Int8Linear,
                   "so3lr_feed_forward": _FeedForward, "so3lr_feed_forward_backward": _FeedForwardBackward}
        calls = {}
        for name, args in plain.items():
            calls[args] = getattr(lib, name), None
            calls[args][0].argtypes = [C.POINTER(args), _p, _p, C.c_size_t]
        for name, args in scratch.items():
            calls[args] = getattr(lib, name), getattr(lib, name + "_workspace")
            calls[args][0].argtypes = [C.POINTER(args), _p, _ll, _p, _p, C.c_size_t]
            calls[args][1].argtypes, calls[args][1].restype = [C.POINTER(args)], _ll
        _CALLS.update(calls)
    return lib


# the current stream's handle without the Stream object that torch.cuda.current_stream makes (2 us)
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _queue(args, like: torch.Tensor) -> None:
    """The C call of `args` on the current stream of like's device, made this thread's device for it."""
    index = like.get_device()
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return _queue(args, like)
    try:
        call, size = _CALLS[type(args)]
        err = _LOCAL.err
    except (KeyError, AttributeError):
        _lib()
        call, size = _CALLS[type(args)]
        err = _LOCAL.err = C.create_string_buffer(_ERR_BYTES)
    if size is None:
        rc = call(args, _raw_stream(index), err, _ERR_BYTES)
    else:
        need = size(args)
        if need > 0:
            ws = like.new_empty(need, dtype=torch.uint8)
            rc = call(args, ws.data_ptr(), need, _raw_stream(index), err, _ERR_BYTES)
        else:
            rc = call(args, None, 0, _raw_stream(index), err, _ERR_BYTES)
    if rc != 0:
        raise So3lrError(err.value.decode(errors="replace") or f"status {rc}")


def _rows(t: torch.Tensor, what: str, like=None, dtype=None, width=None, rows=None) -> torch.Tensor:
    """`t` as a 2-D view of rows with a contiguous last dimension, checked."""
    if not isinstance(t, torch.Tensor) or t.dim() < 1:
        raise ValueError(f"{what} must be a tensor with at least one dimension")
    if not t.is_cuda:
        raise ValueError(f"{what} must be on a CUDA device, got {t.device} (there is no CPU path)")
    if like is not None and t.get_device() != like.get_device():
        raise ValueError(f"{what} is on {t.device}, the other tensors are on {like.device}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, got {t.dtype}")
    if t.dim() != 2:
        t = t.unsqueeze(0) if t.dim() == 1 else t.flatten(0, -2) if t.is_contiguous() else _fold(t, what)
    n, w = t.shape
    if width is not None and w != width:
        raise ValueError(f"{what} must have rows of {width} elements, got {w}")
    if rows is not None and n != rows:
        raise ValueError(f"{what} must have {rows} rows, got {n}")
    if w < 1:
        raise ValueError(f"{what} must have rows of at least one element")
    if t.stride(1) != 1 and w != 1:
        raise ValueError(f"{what} must have a contiguous last dimension")
    return t


def _fold(t: torch.Tensor, what: str) -> torch.Tensor:
    try:
        return t.view(-1, t.shape[-1])
    except RuntimeError:
        raise ValueError(f"the leading dimensions of {what} cannot be seen as rows of one stride") from None


def _dense_rows(t):
    """A gradient as autograd hands it over (expanded, transposed) with the layout the calls take."""
    return t if t is None or t.is_contiguous() else t.contiguous()


def _vector(t: torch.Tensor, what: str, like, dtype, length: int, or_dtype=None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.shape != (length,) or t.get_device() != like.get_device():
        raise ValueError(f"{what} must be a 1-D tensor of {length} elements on {like.device}")
    if t.dtype != dtype and t.dtype != or_dtype:
        raise ValueError(f"{what} must be {dtype}{f' or {or_dtype}' if or_dtype else ''}, got {t.dtype}")
    if length > 1 and t.stride(0) != 1:
        raise ValueError(f"{what} must be contiguous")
    return t


def _type_of(t: torch.Tensor, what: str, types=_TYPES) -> int:
    code = types.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} must be one of {', '.join(map(str, types))}, got {t.dtype}")
    return code


def _codes_like(like: torch.Tensor, rows: int, width: int) -> torch.Tensor:
    """8-bit rows that start on 16-byte boundaries, as int8_linear reads them without a copy."""
    if width % 16 == 0:
        return like.new_empty((rows, width), dtype=torch.int8)
    return like.new_empty((rows, (width + 15) // 16 * 16), dtype=torch.int8)[:, :width]


def _shaped(t: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    return t if like.dim() == 2 else t.view(like.shape[:-1] + t.shape[1:])


# ------------------------------------------------------------------------ norm
def _norm(x, weight, residual, eps, quantize):
    x2 = _rows(x, "x")
    rows, width = x2.shape
    t = _type_of(x2, "x")
    _vector(weight, "weight", x2, x2.dtype, width, torch.float32)
    r_ptr, r_stride, s, s_ptr = None, 0, x, None
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual must have the shape of x, {tuple(x.shape)}, got {tuple(residual.shape)}")
        r2 = _rows(residual, "residual", x2, x2.dtype)
        s = x2.new_empty((rows, width))
        r_ptr, r_stride, s_ptr = r2.data_ptr(), r2.stride(0), s.data_ptr()
        s = _shaped(s, x)
    if quantize:
        y, scales = _codes_like(x2, rows, width), x2.new_empty(rows, dtype=torch.float32)
        out = (None, 0, y.data_ptr(), y.stride(0), scales.data_ptr())
    else:
        y, scales = x2.new_empty((rows, width)), None
        out = (y.data_ptr(), width, None, 0, None)
    if rows:
        _queue(_RmsNorm(rows, width, t, _TYPES[weight.dtype], eps, x2.data_ptr(), x2.stride(0), r_ptr, r_stride,
                        weight.data_ptr(), s_ptr, width, *out), x2)
    return y, scales, s


class _NormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, _, s = _norm(x, weight, residual, eps, False)
        ctx.set_materialize_grads(False)  # an output that nothing reads has no gradient, rather than zeros
        ctx.save_for_backward(s, weight)
        ctx.eps, ctx.has_residual = eps, residual is not None
        return _shaped(y, x), s.view_as(s) if residual is None else s

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, ds):
        s, weight = ctx.saved_tensors
        if dy is None:
            return ds, None, ds if ctx.has_residual else None, None
        dx, dw = rms_norm_backward(_dense_rows(dy), s, weight, _dense_rows(ds), eps=ctx.eps)
        return dx, dw, dx if ctx.has_residual else None, None


def rms_norm(x, weight, residual=None, *, eps: float = 1e-6):
    """(y, s): s = x + residual rounded to x's type (x itself without a
    residual), y = s * weight / sqrt(mean(s^2) + eps). weight: x's type or float32."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (residual is not None and residual.requires_grad)):
        return _NormFunction.apply(x, weight, residual, eps)
    y, _, s = _norm(x, weight, residual, eps, False)
    return _shaped(y, x), s


def rms_norm_int8(x, weight, residual=None, *, eps: float = 1e-6):
    """(codes, scales, s): rms_norm's y in 8 bits, y ~ codes * scales[:, None] with
    scales = max|y| / 127 of each row (float32). Row starts of `codes` are 16-byte aligned."""
    return _norm(x, weight, residual, eps, True)


def rms_norm_backward(dy, s, weight, ds=None, *, eps: float = 1e-6):
    """(dx, dweight) of rms_norm for the gradient dy of y and, optionally, ds that
    of s; dx is also the residual's gradient."""
    s2 = _rows(s, "s")
    rows, width = s2.shape
    t = _type_of(s2, "s")
    _vector(weight, "weight", s2, s2.dtype, width, torch.float32)
    d2 = _rows(dy, "dy", s2, s2.dtype, width, rows)
    e_ptr, e_stride = None, 0
    if ds is not None:
        e2 = _rows(ds, "ds", s2, s2.dtype, width, rows)
        e_ptr, e_stride = e2.data_ptr(), e2.stride(0)
    dx, dw = s2.new_empty((rows, width)), torch.empty_like(weight)
    _queue(_RmsNormBackward(rows, width, t, _TYPES[weight.dtype], eps, d2.data_ptr(), d2.stride(0), s2.data_ptr(),
                            s2.stride(0), weight.data_ptr(), e_ptr, e_stride, dx.data_ptr(), width, dw.data_ptr()), s2)
    return _shaped(dx, s), dw


# ----------------------------------------------------------------------- 8 bits
def int8_linear(a, a_scales, b, b_scales, bias=None, *, out_dtype=torch.bfloat16):
    """y = (a @ b.T) * a_scales[:, None] * b_scales + bias with an int32 sum: a
    [..., k] and b [n, k] int8, scales and bias float32, y [..., n] of out_dtype."""
    a2 = _rows(a, "a", dtype=torch.int8)
    rows, k = a2.shape
    b2 = _rows(b, "b", a2, torch.int8, k)
    n = b2.shape[0]
    t = _TYPES.get(out_dtype)
    if t is None:
        raise ValueError(f"out_dtype must be one of {', '.join(map(str, _TYPES))}, got {out_dtype}")
    _vector(a_scales, "a_scales", a2, torch.float32, rows)
    _vector(b_scales, "b_scales", a2, torch.float32, n)
    if bias is not None:
        _vector(bias, "bias", a2, torch.float32, n)
    if n < 1:
        raise ValueError("b must have at least one row")
    y = a2.new_empty((rows, n), dtype=out_dtype)
    if rows:
        _queue(_Int8Linear(rows, n, k, t, a2.data_ptr(), a2.stride(0), a_scales.data_ptr(), b2.data_ptr(),
                           b2.stride(0), b_scales.data_ptr(), None if bias is None else bias.data_ptr(),
                           y.data_ptr(), n), a2)
    return _shaped(y, a)


def gate_int8(gu):
    """(codes, scales) of silu(g) * u, gu = [g | u] along the last dimension."""
    x = _rows(gu, "gu")
    t = _type_of(x, "gu")
    rows, width = x.shape
    if width % 2:
        raise ValueError(f"gu must hold g and u side by side: an even width, got {width}")
    codes, scales = _codes_like(x, rows, width // 2), x.new_empty(rows, dtype=torch.float32)
    if rows:
        _queue(_GateInt8(rows, width // 2, t, x.data_ptr(), x.stride(0), codes.data_ptr(), codes.stride(0),
                         scales.data_ptr()), x)
    return codes, scales


def dequantize_int8(codes, scales, dtype=torch.bfloat16):
    """codes * scales[:, None], rounded to dtype."""
    c = _rows(codes, "codes", dtype=torch.int8)
    rows, width = c.shape
    t = _TYPES.get(dtype)
    if t is None:
        raise ValueError(f"dtype must be one of {', '.join(map(str, _TYPES))}, got {dtype}")
    _vector(scales, "scales", c, torch.float32, rows)
    out = c.new_empty((rows, width), dtype=dtype)
    if rows:
        _queue(_DequantizeInt8(rows, width, t, c.data_ptr(), c.stride(0), scales.data_ptr(), out.data_ptr(), width), c)
    return _shaped(out, codes)


def quantize_weight(w):
    """(codes, scales) of a weight [n, k], a scale for each output channel: done
    once when a model is loaded, with the same rounding as rms_norm_int8."""
    w2 = _rows(w, "w")
    _type_of(w2, "w")
    f = w2.detach().float()
    scales = f.abs().amax(1) / 127.0
    codes = _codes_like(w2, *w2.shape)
    codes.copy_(torch.round(f / torch.where(scales > 0, scales, 1.0)[:, None]).clamp_(-127, 127))
    return codes, scales


# ----------------------------------------------------------------- feed-forward
def _ffn_operands(x, w_gate, w_up, w_down):
    x2 = _rows(x, "x")
    t = _type_of(x2, "x", _HALF)
    width, dtype = x2.shape[1], x2.dtype
    g = _rows(w_gate, "w_gate", x2, dtype, width)
    hidden = g.shape[0]
    if hidden < 1:
        raise ValueError("w_gate must have at least one row")
    u = _rows(w_up, "w_up", x2, dtype, width, hidden)
    d = _rows(w_down, "w_down", x2, dtype, hidden, width)
    return x2, t, hidden, (x2.data_ptr(), x2.stride(0), g.data_ptr(), g.stride(0), u.data_ptr(), u.stride(0),
                           d.data_ptr(), d.stride(0))


def _ffn(x, w_gate, w_up, w_down, keep=False):
    x2, t, hidden, operands = _ffn_operands(x, w_gate, w_up, w_down)
    rows, width = x2.shape
    y = x2.new_empty((rows, width))
    h = x2.new_empty((rows, hidden)) if keep else None
    if rows:
        _queue(_FeedForward(rows, width, hidden, t, *operands, y.data_ptr(), width, h.data_ptr() if keep else None), x2)
    return _shaped(y, x), h


class _FeedForwardFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down):
        y, saved = feed_forward_train(x, w_gate, w_up, w_down)
        ctx.save_for_backward(*saved)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return feed_forward_backward(_dense_rows(dy), ctx.saved_tensors)


def feed_forward(x, w_gate, w_up, w_down):
    """y = (silu(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T, bfloat16 or float16:
    x [..., width], w_gate and w_up [hidden, width], w_down [width, hidden]."""
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad or
                                    w_down.requires_grad):
        return _FeedForwardFunction.apply(x, w_gate, w_up, w_down)
    return _ffn(x, w_gate, w_up, w_down)[0]


def feed_forward_train(x, w_gate, w_up, w_down):
    """(y, saved): feed_forward, and what feed_forward_backward needs of it."""
    y, h = _ffn(x, w_gate, w_up, w_down, keep=True)
    return y, (x, w_gate, w_up, w_down, h)


def feed_forward_backward(dy, saved):
    """(dx, dw_gate, dw_up, dw_down) for the gradient dy of feed_forward_train's y."""
    x, w_gate, w_up, w_down, h = saved
    x2, t, hidden, operands = _ffn_operands(x, w_gate, w_up, w_down)
    rows, width = x2.shape
    d2 = _rows(dy, "dy", x2, x2.dtype, width, rows)
    if h.shape != (rows, hidden) or h.dtype != x2.dtype or not h.is_contiguous():
        raise ValueError("saved does not come from feed_forward_train")
    dx = x2.new_empty((rows, width))
    dwg, dwu, dwd = x2.new_empty((hidden, width)), x2.new_empty((hidden, width)), x2.new_empty((width, hidden))
    _queue(_FeedForwardBackward(rows, width, hidden, t, d2.data_ptr(), d2.stride(0), *operands, h.data_ptr(),
                                dx.data_ptr(), width, dwg.data_ptr(), dwu.data_ptr(), dwd.data_ptr()), x2)
    return _shaped(dx, x), dwg, dwu, dwd


# ------------------------------------------------------------------ the sublayer
class FeedForwardBlock(torch.nn.Module):
    """Pre-norm gated feed-forward sublayer over rows of features:

        y, s = rms_norm(x, norm, residual);  out = feed_forward(y, w_gate, w_up, w_down)

    forward(x, residual) returns (out, s): the next block adds `out` to the
    stream `s`. Trains through autograd."""

    def __init__(self, width: int, hidden: int, *, eps: float = 1e-6, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        self.eps = eps
        make = lambda *shape: torch.nn.Parameter(  # noqa: E731
            torch.randn(*shape, device=device).mul_(shape[1] ** -0.5).to(dtype))
        self.norm = torch.nn.Parameter(torch.ones(width, device=device))
        self.w_gate, self.w_up, self.w_down = make(hidden, width), make(hidden, width), make(width, hidden)

    def forward(self, x, residual=None):
        y, s = rms_norm(x, self.norm, residual, eps=self.eps)
        return feed_forward(y, self.w_gate, self.w_up, self.w_down), s


class Int8FeedForwardBlock:
    """A FeedForwardBlock's weights served in 8 bits: the same call and shapes,
    no gradients. Weights are put into 8 bits once, activations row by row."""

    def __init__(self, block: FeedForwardBlock):
        self.eps, self.dtype = block.eps, block.w_down.dtype
        self.norm = block.norm.detach().clone()
        self.gate_up = quantize_weight(torch.cat([block.w_gate.detach(), block.w_up.detach()]))
        self.down = quantize_weight(block.w_down)

    @torch.no_grad()
    def __call__(self, x, residual=None):
        codes, scales, s = rms_norm_int8(x, self.norm, residual, eps=self.eps)
        gu = int8_linear(codes, scales, *self.gate_up, out_dtype=self.dtype)
        codes, scales = gate_int8(gu)
        out = int8_linear(codes, scales, *self.down, out_dtype=self.dtype)
        return out.view(x.shape), s
