"""C entry points of the row-wise feed-forward layers: every refusal happens on the
host, before any CUDA call, with a message. No GPU."""
import ctypes as C

import pytest

pytest.importorskip("torch")


@pytest.fixture(scope="module")
def layers():
    from so3lr_b200 import layers
    layers._lib()
    return layers


def _refused(layers, name, args, message, workspace=None):
    err = C.create_string_buffer(512)
    fn = getattr(layers._lib(), name)
    rc = fn(args, *workspace, None, err, 512) if workspace is not None else fn(args, None, err, 512)
    assert rc != 0 and message in err.value.decode(), err.value


def _norm(layers, **kw):
    a = layers._RmsNorm(rows=2, width=8, dtype=1, weight_dtype=0, eps=1e-6, x=4096, x_stride=8, weight=4096, y=4096,
                        y_stride=8)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change, message", [
    (dict(rows=-1), "rows must be in"), (dict(width=0), "width must be in"), (dict(width=16385), "width must be in"),
    (dict(dtype=3), "dtype must be"), (dict(weight_dtype=2), "weight_dtype must be"), (dict(eps=-1.0), "eps must be"),
    (dict(eps=float("nan")), "eps must be"), (dict(x=None), "x is NULL"), (dict(x=4097), "x is not aligned"),
    (dict(x_stride=-8), "x needs a row stride"), (dict(weight=None), "weight is NULL"), (dict(y=None), "exactly one"),
    (dict(codes=4096, codes_stride=8), "exactly one"), (dict(y_stride=7), "y needs a row stride of at least"),
    (dict(residual=4096), "s must be given"), (dict(s=4096), "s must be given"),
    (dict(residual=4096, residual_stride=8, s=4096, s_stride=4), "s needs a row stride of at least"),
    (dict(y=None, codes=4096, codes_stride=8), "scales is NULL"),
])
def test_rms_norm_refusals(layers, change, message):
    _refused(layers, "so3lr_rms_norm", _norm(layers, **change), message)


def test_null_arguments(layers):
    for name in ("so3lr_rms_norm", "so3lr_gate_int8", "so3lr_dequantize_int8"):
        _refused(layers, name, None, "args is NULL")
    for name in ("so3lr_rms_norm_backward", "so3lr_int8_linear", "so3lr_feed_forward", "so3lr_feed_forward_backward"):
        _refused(layers, name, None, "args is NULL", workspace=(None, 0))
        assert getattr(layers._lib(), name + "_workspace")(None) == -1
    # without a message buffer too
    assert layers._lib().so3lr_rms_norm(None, None, None, 0) != 0


@pytest.mark.parametrize("change, message", [
    (dict(rows=1 << 40), "rows must be in"), (dict(k=131072), "k must be in"), (dict(n=0), "n must be in"),
    (dict(out_dtype=-1), "out_dtype must be"), (dict(a=None), "a is NULL"), (dict(b_scales=None), "b_scales is NULL"),
    (dict(a_scales=4098), "a_scales is not aligned"), (dict(y_stride=3), "y needs a row stride of at least"),
])
def test_int8_linear_refusals(layers, change, message):
    a = layers._Int8Linear(rows=2, n=4, k=8, out_dtype=0, a=4096, a_stride=8, a_scales=4096, b=4096, b_stride=8,
                           b_scales=4096, y=4096, y_stride=4)
    for k, v in change.items():
        setattr(a, k, v)
    _refused(layers, "so3lr_int8_linear", a, message, workspace=(4096, 1 << 40))


@pytest.mark.parametrize("change, message", [
    (dict(dtype=0), "must be SO3LR_BFLOAT16 or SO3LR_FLOAT16"), (dict(hidden=0), "hidden must be in"),
    (dict(x=None), "x is NULL"), (dict(w_gate=4097), "w_gate is not aligned"), (dict(w_down=None), "w_down is NULL"),
    (dict(y_stride=1), "y needs a row stride of at least"),
])
def test_feed_forward_refusals(layers, change, message):
    a = layers._FeedForward(rows=2, width=8, hidden=16, dtype=1, x=4096, x_stride=8, w_gate=4096, w_gate_stride=8,
                            w_up=4096, w_up_stride=8, w_down=4096, w_down_stride=16, y=4096, y_stride=8)
    for k, v in change.items():
        setattr(a, k, v)
    _refused(layers, "so3lr_feed_forward", a, message, workspace=(4096, 1 << 40))


def test_workspaces_are_checked(layers):
    a = layers._FeedForward(rows=200, width=64, hidden=128, dtype=1, x=4096, x_stride=64, w_gate=4096,
                            w_gate_stride=64, w_up=4096, w_up_stride=64, w_down=4096, w_down_stride=128, y=4096,
                            y_stride=64)
    need = layers._lib().so3lr_feed_forward_workspace(a)
    assert need > 0
    _refused(layers, "so3lr_feed_forward", a, "bytes, ", workspace=(4096, need - 1))
    _refused(layers, "so3lr_feed_forward", a, "workspace is NULL", workspace=(None, need))
    _refused(layers, "so3lr_feed_forward", a, "workspace is not aligned", workspace=(4096 + 16, need))
    a.hidden = -5
    assert layers._lib().so3lr_feed_forward_workspace(a) == -1


def test_cpu_tensors_are_refused(layers):
    import torch
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="there is no CPU path"):
        layers.rms_norm(x, torch.ones(64))
    with pytest.raises(ValueError, match="there is no CPU path"):
        layers.feed_forward(x, x, x, x)
