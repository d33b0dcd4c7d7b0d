"""C entry points of the row-wise feed-forward layers: every refusal happens on the
host, before any CUDA call, with a message. No GPU."""
import ctypes as C

import pytest

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
                ("w_down_stride", _ll), ("y", _p), ("y_stride", _ll), ("h", _p), ("gu", _p)]


class _FeedForwardBackward(C.Structure):
    _fields_ = [("rows", _ll), ("width", _ll), ("hidden", _ll), ("dtype", _i), ("dy", _p), ("dy_stride", _ll),
                ("x", _p), ("x_stride", _ll), ("w_gate", _p), ("w_gate_stride", _ll), ("w_up", _p),
                ("w_up_stride", _ll), ("w_down", _p), ("w_down_stride", _ll), ("h", _p), ("gu", _p), ("dx", _p), ("dx_stride", _ll),
                ("dw_gate", _p), ("dw_up", _p), ("dw_down", _p)]


@pytest.fixture(scope="module")
def lib():
    """The library with the layers' argument types declared."""
    from so3lr_b200 import load_library
    lib = load_library()
    for name, args in {"so3lr_rms_norm": _RmsNorm, "so3lr_gate_int8": _GateInt8,
                       "so3lr_dequantize_int8": _DequantizeInt8}.items():
        getattr(lib, name).argtypes = [C.POINTER(args), _p, _p, C.c_size_t]
    for name, args in {"so3lr_rms_norm_backward": _RmsNormBackward, "so3lr_int8_linear": _Int8Linear,
                       "so3lr_feed_forward": _FeedForward, "so3lr_feed_forward_backward": _FeedForwardBackward}.items():
        getattr(lib, name).argtypes = [C.POINTER(args), _p, _ll, _p, _p, C.c_size_t]
        size = getattr(lib, name + "_workspace")
        size.argtypes, size.restype = [C.POINTER(args)], _ll
    lib.so3lr_feed_forward_keep.argtypes, lib.so3lr_feed_forward_keep.restype = [C.POINTER(_FeedForward)], _ll
    return lib


def _refused(lib, name, args, message, workspace=None):
    err = C.create_string_buffer(512)
    fn = getattr(lib, name)
    rc = fn(args, *workspace, None, err, 512) if workspace is not None else fn(args, None, err, 512)
    assert rc != 0 and message in err.value.decode(), err.value


def _norm(**kw):
    a = _RmsNorm(rows=2, width=8, dtype=1, weight_dtype=0, eps=1e-6, x=4096, x_stride=8, weight=4096, y=4096,
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
def test_rms_norm_refusals(lib, change, message):
    _refused(lib, "so3lr_rms_norm", _norm(**change), message)


def test_null_arguments(lib):
    for name in ("so3lr_rms_norm", "so3lr_gate_int8", "so3lr_dequantize_int8"):
        _refused(lib, name, None, "args is NULL")
    for name in ("so3lr_rms_norm_backward", "so3lr_int8_linear", "so3lr_feed_forward", "so3lr_feed_forward_backward"):
        _refused(lib, name, None, "args is NULL", workspace=(None, 0))
        assert getattr(lib, name + "_workspace")(None) == -1
    # without a message buffer too
    assert lib.so3lr_rms_norm(None, None, None, 0) != 0


@pytest.mark.parametrize("change, message", [
    (dict(rows=1 << 40), "rows must be in"), (dict(k=131072), "k must be in"), (dict(n=0), "n must be in"),
    (dict(out_dtype=-1), "out_dtype must be"), (dict(a=None), "a is NULL"), (dict(b_scales=None), "b_scales is NULL"),
    (dict(a_scales=4098), "a_scales is not aligned"), (dict(y_stride=3), "y needs a row stride of at least"),
])
def test_int8_linear_refusals(lib, change, message):
    a = _Int8Linear(rows=2, n=4, k=8, out_dtype=0, a=4096, a_stride=8, a_scales=4096, b=4096, b_stride=8,
                           b_scales=4096, y=4096, y_stride=4)
    for k, v in change.items():
        setattr(a, k, v)
    _refused(lib, "so3lr_int8_linear", a, message, workspace=(4096, 1 << 40))


@pytest.mark.parametrize("change, message", [
    (dict(dtype=0), "must be SO3LR_BFLOAT16 or SO3LR_FLOAT16"), (dict(hidden=0), "hidden must be in"),
    (dict(x=None), "x is NULL"), (dict(w_gate=4097), "w_gate is not aligned"), (dict(w_down=None), "w_down is NULL"),
    (dict(y_stride=1), "y needs a row stride of at least"),
])
def test_feed_forward_refusals(lib, change, message):
    a = _FeedForward(rows=2, width=8, hidden=16, dtype=1, x=4096, x_stride=8, w_gate=4096, w_gate_stride=8,
                            w_up=4096, w_up_stride=8, w_down=4096, w_down_stride=16, y=4096, y_stride=8)
    for k, v in change.items():
        setattr(a, k, v)
    _refused(lib, "so3lr_feed_forward", a, message, workspace=(4096, 1 << 40))


def test_workspaces_are_checked(lib):
    a = _FeedForward(rows=500, width=64, hidden=128, dtype=1, x=4096, x_stride=64, w_gate=4096,
                            w_gate_stride=64, w_up=4096, w_up_stride=64, w_down=4096, w_down_stride=128, y=4096,
                            y_stride=64)
    need = lib.so3lr_feed_forward_workspace(a)
    assert need > 0
    _refused(lib, "so3lr_feed_forward", a, "bytes, ", workspace=(4096, need - 1))
    _refused(lib, "so3lr_feed_forward", a, "workspace is NULL", workspace=(None, need))
    _refused(lib, "so3lr_feed_forward", a, "workspace is not aligned", workspace=(4096 + 16, need))
    a.hidden = -5
    assert lib.so3lr_feed_forward_workspace(a) == -1


def test_projections_are_kept_for_wide_layers(lib):
    """Nothing for narrow layers or a few rows; else whole blocks of 32 rows of two float32 values."""
    a = _FeedForward(rows=1000, width=4096, hidden=24, dtype=1)
    assert lib.so3lr_feed_forward_keep(a) == 1024 * 24 * 2 * 4
    a.rows = 1
    assert lib.so3lr_feed_forward_keep(a) == 0
    a.rows, a.width = 1000, 64
    assert lib.so3lr_feed_forward_keep(a) == 0
    a.width = 0
    assert lib.so3lr_feed_forward_keep(a) == -1


def test_cpu_tensors_are_refused():
    torch = pytest.importorskip("torch")
    from so3lr_b200 import layers
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="there is no CPU path"):
        layers.rms_norm(x, torch.ones(64))
    with pytest.raises(ValueError, match="there is no CPU path"):
        layers.feed_forward(x, x, x, x)
    with pytest.raises(ValueError, match="x must be a tensor"):
        layers._layers.feed_forward(None, x, x, x, False)
    with pytest.raises(TypeError):
        layers._layers.gate_int8()
