"""C entry points of the dense layer and of the norms on both sides of a block: every refusal
happens on the host, before any CUDA call, with a message. No GPU."""
import ctypes as C
import pathlib
import re

import pytest

_ll, _p, _i, _d = C.c_longlong, C.c_void_p, C.c_int, C.c_double


def _structure(spec):
    types = dict(l=_ll, p=_p, i=_i, d=_d)
    return type("Args", (C.Structure,), {"_fields_": [(n, types[t]) for n, t in (f.split(":") for f in spec.split())]})


_Linear = _structure("rows:l n:l k:l dtype:i bias_dtype:i activation:i x:p x_stride:l w:p w_stride:l bias:p residual:p "
                     "residual_stride:l y:p y_stride:l z:p z_stride:l")
_LinearBackward = _structure("rows:l n:l k:l dtype:i bias_dtype:i activation:i dy:p dy_stride:l x:p x_stride:l w:p w_stride:l "
                             "z:p z_stride:l dx:p dx_stride:l dw:p dbias:p")
_Sandwich = _structure("rows:l width:l dtype:i weight_dtype:i eps:d x:p x_stride:l residual:p residual_stride:l gate:p "
                       "gate_stride:l weight:p next_weight:p residual_scale:p s:p s_stride:l y:p y_stride:l")
_SandwichBackward = _structure("rows:l width:l dtype:i weight_dtype:i eps:d dy:p dy_stride:l ds:p ds_stride:l s:p s_stride:l "
                               "x:p x_stride:l residual:p residual_stride:l gate:p gate_stride:l weight:p next_weight:p "
                               "residual_scale:p dx:p dx_stride:l dresidual:p dresidual_stride:l dgate:p dgate_stride:l "
                               "dweight:p dnext_weight:p dresidual_scale:p")
CALLS = {"so3lr_linear": _Linear, "so3lr_linear_backward": _LinearBackward, "so3lr_sandwich_norm": _Sandwich,
         "so3lr_sandwich_norm_backward": _SandwichBackward}
NO_WORKSPACE = {"so3lr_sandwich_norm"}


@pytest.fixture(scope="module")
def lib():
    from so3lr_b200 import load_library
    lib = load_library()
    for name, args in CALLS.items():
        scratch = [] if name in NO_WORKSPACE else [_p, _ll]
        getattr(lib, name).argtypes = [C.POINTER(args)] + scratch + [_p, C.c_char_p, C.c_size_t]
        if scratch:
            size = getattr(lib, name + "_workspace")
            size.argtypes, size.restype = [C.POINTER(args)], _ll
    return lib


def _good(name, rows=300):
    """Addresses that are never read: all refusals come first."""
    a = CALLS[name]()
    at = 1 << 20
    for field, kind in a._fields_:
        if kind is _p:
            at += 1 << 24
            setattr(a, field, at)
        elif field.endswith("_stride"):
            setattr(a, field, 264)
    a.rows, a.dtype = rows, 1
    if "linear" in name:
        a.n, a.k, a.bias_dtype, a.activation = 200, 96, 1, 1
    else:
        a.width, a.weight_dtype, a.eps = 256, 0, 1e-6
    return a


def _call(lib, name, a, workspace=256, size=1 << 40):
    err = C.create_string_buffer(1024)
    scratch = [] if name in NO_WORKSPACE else [workspace, size]
    rc = getattr(lib, name)(C.byref(a) if a is not None else None, *scratch, None, err, 1024)
    return rc, err.value.decode()


LINEAR = [(dict(rows=-1), "rows must be in"), (dict(n=0), "n must be in"), (dict(k=(1 << 20) + 1), "k must be in"),
          (dict(dtype=0), "dtype must be"), (dict(dtype=3), "dtype must be"), (dict(bias_dtype=2), "bias_dtype must be"),
          (dict(activation=-1), "activation must be"), (dict(activation=5), "activation must be"), (dict(x=None), "x is NULL"),
          (dict(w=3), "w is not aligned"), (dict(x_stride=-1), "x needs a row stride"), (dict(z=5), "z is not aligned")]
SANDWICH = [(dict(rows=1 << 31), "rows must be in"), (dict(width=16385), "width must be in"), (dict(width=0), "width must be in"),
            (dict(dtype=7), "dtype must be"), (dict(weight_dtype=2), "weight_dtype must be"), (dict(eps=-1.0), "eps must be"),
            (dict(eps=float("nan")), "eps must be"), (dict(x=None), "x is NULL"), (dict(gate=1), "gate is not aligned"),
            (dict(gate_stride=-2), "gate needs a row stride"), (dict(weight=None), "weight is NULL"),
            (dict(next_weight=2), "next_weight is not aligned"), (dict(residual_scale=2), "residual_scale is not aligned"),
            (dict(s=None), "s is NULL")]
CASES = ([("so3lr_linear", *c) for c in LINEAR + [
             (dict(y=None), "y is NULL"), (dict(y_stride=199), "y needs a row stride of at least"),
             (dict(residual=7), "residual is not aligned"), (dict(bias=1), "bias is not aligned"),
             (dict(z_stride=5), "z needs a row stride of at least")]]
         + [("so3lr_linear_backward", *c) for c in LINEAR + [
             (dict(dy=None), "dy is NULL"), (dict(z=None), "z is NULL"), (dict(dx_stride=95), "dx needs a row stride of at least"),
             (dict(dw=1), "dw is not aligned"), (dict(dbias=1), "dbias is not aligned")]]
         + [("so3lr_sandwich_norm", *c) for c in SANDWICH + [
             (dict(residual=None), "residual is NULL"), (dict(y_stride=255), "y needs a row stride of at least")]]
         + [("so3lr_sandwich_norm_backward", *c) for c in SANDWICH + [
             (dict(dy=None), "dy is NULL"), (dict(residual=None), "residual is NULL"), (dict(dgate=None), "dgate must be given"),
             (dict(gate=None), "dgate must be given"), (dict(dresidual_scale=None), "dresidual_scale must be given"),
             (dict(residual_scale=None), "dresidual_scale must be given"), (dict(dresidual_stride=3), "dresidual needs a row stride"),
             (dict(dnext_weight=None), "dnext_weight is NULL"), (dict(ds=1), "ds is not aligned")]])


@pytest.mark.parametrize("name, change, said", CASES)
def test_refusals(lib, name, change, said):
    a = _good(name)
    for k, v in change.items():
        assert hasattr(a, k)
        setattr(a, k, v)
    rc, err = _call(lib, name, a)
    assert rc == 1 and err.startswith(name) and said in err, err


@pytest.mark.parametrize("name", sorted(CALLS))
def test_no_arguments_and_workspaces(lib, name):
    rc, err = _call(lib, name, None)
    assert rc == 1 and "args is NULL" in err
    if name in NO_WORKSPACE:
        return
    size = getattr(lib, name + "_workspace")
    a = _good(name, rows=40000)
    need = size(C.byref(a))
    assert need >= 0 and size(None) == -1
    bad = _good(name)
    bad.dtype = 9
    assert size(C.byref(bad)) == -1
    if need:
        for workspace, have, said in ((256, need - 1, "the workspace has"), (None, need, "workspace is NULL"),
                                      (128, need, "workspace is not aligned")):
            rc, err = _call(lib, name, a, workspace, have)
            assert rc == 1 and said in err, err


def test_no_rows_is_no_work(lib):
    for name in ("so3lr_linear", "so3lr_sandwich_norm"):
        a = _good(name, rows=0)
        assert _call(lib, name, a) == (0, "")


def test_fields_are_the_header_s():
    """The structures of this file name the header's fields in its order."""
    header = (pathlib.Path(__file__).resolve().parents[1] / "include" / "so3lr_b200.h").read_text()
    header = re.sub(r"/\*.*?\*/", "", header, flags=re.S)
    for name, args in CALLS.items():
        body = re.search(r"typedef struct \{([^}]*)\} %s_args;" % name, header).group(1)
        names = [w.strip().lstrip("*") for line in body.split(";") for w in re.sub(r"^\s*(const )?(long long|int|double|void|float)", "", line.strip()).split(",")]
        assert [n for n in names if n] == [f for f, _ in args._fields_], name


@pytest.mark.parametrize("name", ["adamw.cu", "sandwich.cu", "linear.cu", "activation.cuh", "row_team.cuh"])
def test_no_read_only_loads(name):
    """Kernels that start while the kernel before them may still write what they read promise
    nothing of it: no non-coherent loads, by name or by a pointer to const without alias."""
    text = (pathlib.Path(__file__).resolve().parents[1] / "so3lr_b200" / "csrc" / name).read_text()
    code = re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)
    assert not re.search(r"\.nc\b|__ldg\s*\(|\bconst\b[^,;()]*\*\s*__restrict__", code)
