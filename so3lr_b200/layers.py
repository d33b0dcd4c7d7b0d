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

``rms_norm`` and ``feed_forward`` record themselves for reverse-mode autograd when an
argument requires a gradient; tensors with a forward-mode tangent and
``torch.jit.trace`` are refused. All other calls record nothing: their results, the
stream of ``rms_norm_int8`` among them, are detached from arguments that require a
gradient. ``FeedForwardBlock`` and ``Int8FeedForwardBlock`` run them
together: the pre-norm sublayer as it is trained, and the same weights served
in 8 bits.

The calls are the entry points of include/so3lr_b200.h ("Row-wise feed-forward
layers") through the compiled module ``so3lr_b200._layers``
(binding/layers_binding.cpp): they queue kernels on the current torch stream of the
tensors' GPU and return; outputs and scratch come from torch's allocator. A kernel
whose wait gives up is reported by the next call on that GPU and by ``check_status``.
Rows are all leading dimensions; the last dimension must be contiguous, rows may have
any stride. Arguments that do not fit one another raise ValueError; a length or an eps
outside the library's range, and failures of the library, So3lrError. There is no CPU
path: a tensor that is not on a GPU is refused.
"""
from __future__ import annotations

import torch

from .runtime import So3lrError, load_library

try:
    load_library()
    from . import _layers
except (ImportError, So3lrError) as e:
    raise ImportError(f"the feed-forward layers' module is missing or does not fit the installed torch ({e}): build it "
                      "with `python -m so3lr_b200.build`, which needs a torch with CUDA and Python's headers") from e

__all__ = ["rms_norm", "rms_norm_int8", "rms_norm_backward", "int8_linear", "gate_int8", "dequantize_int8",
           "quantize_weight", "feed_forward", "feed_forward_train", "feed_forward_backward", "FeedForwardBlock",
           "Int8FeedForwardBlock", "check_status", "set_wait_limit"]


def check_status(device=None) -> None:
    """Raises So3lrError if a kernel of an earlier call on `device` (the current one by
    default) gave up waiting: the results of that call and of those after it are not
    valid. Calls on the device are refused from then on until this has said so, once.
    It does not synchronise: ask after doing so to know about the last calls too."""
    index = None if device is None else torch.device(device).index
    _layers.status(torch.cuda.current_device() if index is None else index)


def set_wait_limit(cycles: int = 0) -> None:
    """About how many clock cycles of an SM a wait inside the kernels that are queued
    from now on may take; 0: the default of 4e9, about 2 s."""
    _layers.set_wait_limit(cycles)


def _dense_rows(t):
    """A gradient as autograd hands it over (expanded, transposed) with the layout the calls take."""
    return t if t is None or t.is_contiguous() else t.contiguous()


# ------------------------------------------------------------------------ norm
class _NormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, _, s = _layers.rms_norm(x, weight, residual, eps, False)
        ctx.set_materialize_grads(False)  # an output that nothing reads has no gradient, rather than zeros
        ctx.save_for_backward(s, weight)
        ctx.eps, ctx.has_residual = eps, residual is not None
        return y, s.view_as(s) if residual is None else s

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, ds):
        s, weight = ctx.saved_tensors
        if dy is None:
            return ds, None, ds if ctx.has_residual else None, None
        dx, dw = _layers.rms_norm_backward(_dense_rows(dy), s, weight, _dense_rows(ds), ctx.eps)
        return dx, dw, dx if ctx.has_residual else None, None


def rms_norm(x, weight, residual=None, *, eps: float = 1e-6):
    """(y, s): s = x + residual rounded to x's type (x itself, detached under no_grad,
    without a residual), y = s * weight / sqrt(mean(s^2) + eps). weight: x's type or float32."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (residual is not None and residual.requires_grad)):
        return _NormFunction.apply(x, weight, residual, eps)
    y, _, s = _layers.rms_norm(x, weight, residual, eps, False)
    return y, s.detach() if s.requires_grad else s


def rms_norm_int8(x, weight, residual=None, *, eps: float = 1e-6):
    """(codes, scales, s): rms_norm's y in 8 bits, one row for each row of x:
    y ~ codes * scales[:, None] with scales = max|y| / 127 of each row (float32) and
    codes = y / scale rounded to nearest; the quotient is formed with a reciprocal, so
    that a y within a few float32 units of a tie may fall on its other side. Row starts
    of `codes` are 16-byte aligned. Records nothing for autograd: s is detached with a
    residual and without one."""
    codes, scales, s = _layers.rms_norm(x, weight, residual, eps, True)
    return codes, scales, s.detach() if s.requires_grad else s


def rms_norm_backward(dy, s, weight, ds=None, *, eps: float = 1e-6):
    """(dx, dweight) of rms_norm for the gradient dy of y and, optionally, ds that
    of s; dx is also the residual's gradient."""
    return _layers.rms_norm_backward(dy, s, weight, ds, eps)


# ----------------------------------------------------------------------- 8 bits
def int8_linear(a, a_scales, b, b_scales, bias=None, *, out_dtype=torch.bfloat16):
    """y = (a @ b.T) * a_scales[:, None] * b_scales + bias with an int32 sum: a
    [..., k] and b [n, k] int8, scales and bias float32, y [..., n] of out_dtype."""
    return _layers.int8_linear(a, a_scales, b, b_scales, bias, out_dtype)


def gate_int8(gu):
    """(codes, scales) of silu(g) * u, gu = [g | u] along the last dimension."""
    return _layers.gate_int8(gu)


def dequantize_int8(codes, scales, dtype=torch.bfloat16):
    """codes * scales[:, None], rounded to dtype."""
    return _layers.dequantize_int8(codes, scales, dtype)


def quantize_weight(w):
    """(codes, scales) of a weight [n, k], a scale for each output channel: done
    once when a model is loaded. codes = w / scale rounded to nearest, ties to even;
    channels of zeros get scale 0, channels with an infinity or a NaN scale NaN, both
    codes 0. Row starts of `codes` are 16-byte aligned."""
    f = w.detach().float()
    n, k = f.shape
    scales = f.abs().amax(1) / 127.0
    live = scales.isfinite() & (scales > 0)
    quotients = torch.where(live[:, None], f / torch.where(live, scales, 1.0)[:, None], 0.0)
    codes = torch.empty((n, (k + 15) // 16 * 16), dtype=torch.int8, device=f.device)[:, :k]
    codes.copy_(torch.round(quotients).clamp_(-127, 127))
    return codes, torch.where(scales.isfinite(), scales, torch.nan)


# ----------------------------------------------------------------- feed-forward
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
    x [..., width], w_gate and w_up [hidden, width], w_down [width, hidden].

    The hidden layer is rounded to x's type between the products, in calls of few rows
    (16, or up to 256 through small weights) to two such parts: a row's result can
    differ in its last bits between calls of few and of many rows. With autograd the
    operands and the hidden layer are kept, and for widths of 1024 and more and many
    rows the two projections in float32, 8 bytes for each element of the hidden layer
    (537 MB for 8190 rows of 8200). The backward pass computes the gradients of all
    four operands, whichever are asked for."""
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad or
                                    w_down.requires_grad):
        return _FeedForwardFunction.apply(x, w_gate, w_up, w_down)
    return _layers.feed_forward(x, w_gate, w_up, w_down, False)


def feed_forward_train(x, w_gate, w_up, w_down):
    """(y, saved): feed_forward, and what feed_forward_backward needs of it: the
    operands, the hidden layer and, for wide layers, the two projections in float32."""
    y, h, gu = _layers.feed_forward(x, w_gate, w_up, w_down, True)
    return y, (x, w_gate, w_up, w_down, h, gu)


def feed_forward_backward(dy, saved):
    """(dx, dw_gate, dw_up, dw_down) for the gradient dy of feed_forward_train's y."""
    x, w_gate, w_up, w_down, h, gu = saved
    return _layers.feed_forward_backward(x, w_gate, w_up, w_down, dy, h, gu)


# ------------------------------------------------------------------ the sublayer
class FeedForwardBlock(torch.nn.Module):
    """Pre-norm gated feed-forward sublayer over rows of features:

        y, s = rms_norm(x, norm, residual);  out = feed_forward(y, w_gate, w_up, w_down)

    forward(x, residual) returns (out, s): the next block adds `out` to the
    stream `s`. Trains through autograd (see feed_forward for what that keeps)."""

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
