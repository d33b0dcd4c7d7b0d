"""C entry points of the AdamW step: every refusal happens on the host, before any CUDA
call, with a message. No GPU."""
import ctypes as C

import pytest

_ll, _p, _i, _d = C.c_longlong, C.c_void_p, C.c_int, C.c_double


class _Tensor(C.Structure):
    _fields_ = [("param", _p), ("grad", _p), ("master", _p), ("exp_avg", _p), ("exp_avg_sq", _p), ("exp_avg_scale", _p),
                ("exp_avg_sq_scale", _p), ("step", _p), ("n", _ll), ("dtype", _i), ("grad_dtype", _i)]


class _Adamw(C.Structure):
    _fields_ = [("count", _ll), ("tensors", C.POINTER(_Tensor)), ("lr", _d), ("lr_device", _p), ("beta1", _d),
                ("beta2", _d), ("eps", _d), ("weight_decay", _d)]


class _Values(C.Structure):
    _fields_ = [("n", _ll), ("is_signed", _i), ("dtype", _i), ("codes", _p), ("scales", _p), ("values", _p)]


@pytest.fixture(scope="module")
def lib():
    from so3lr_b200 import load_library
    lib = load_library()
    lib.so3lr_adamw.argtypes = [C.POINTER(_Adamw), _p, _ll, _p, C.c_char_p, C.c_size_t]
    lib.so3lr_adamw_workspace.argtypes, lib.so3lr_adamw_workspace.restype = [C.POINTER(_Adamw)], _ll
    lib.so3lr_moment_values.argtypes = [C.POINTER(_Values), _p, C.c_char_p, C.c_size_t]
    return lib


def _args(count=2, **change):
    """Addresses that are never read: all refusals come first."""
    tensors = (_Tensor * max(count, 1))()
    for i in range(count):
        at = 1 << 20 * (i + 1)
        tensors[i] = _Tensor(at, at + 4096, at + 8192, at + 16384, at + 32768, None, None, at + 65536, 100, 1, 1)
    a = _Adamw(count, tensors, 1e-3, None, 0.9, 0.999, 1e-8, 0.01)
    for k, v in change.items():
        if k.startswith("t_"):
            setattr(tensors[0], k[2:], v)
        else:
            setattr(a, k, v)
    a.keep = tensors
    return a


@pytest.mark.parametrize("change, said", [
    (dict(t_param=None), "param is NULL"), (dict(t_param=(1 << 20) + 1), "param is not aligned"),
    (dict(t_grad=None), "grad is NULL"), (dict(t_exp_avg=None), "exp_avg is NULL"),
    (dict(t_exp_avg_sq=6), "exp_avg_sq is not aligned"), (dict(t_step=None), "step is NULL"),
    (dict(t_step=12), "step is not aligned"), (dict(t_n=-1), "n must be in"), (dict(t_n=(1 << 40) + 1), "n must be in"),
    (dict(t_dtype=3), "dtype must be"), (dict(t_grad_dtype=2), "grad_dtype must be"),
    (dict(t_exp_avg_scale=64), "must be given together"), (dict(t_exp_avg_scale=64, t_exp_avg_sq_scale=66), "not aligned"),
    (dict(t_dtype=0, t_grad_dtype=0), "master is for 16-bit"), (dict(t_param=(1 << 40) + 198), "parameters overlap"),
    (dict(t_step=(1 << 40) + 65536), "step counters overlap"), (dict(lr=-1e-3), "lr must be"),
    (dict(lr=float("inf")), "lr must be"), (dict(lr=float("nan")), "lr must be"), (dict(lr_device=2), "lr_device is not aligned"),
    (dict(beta1=1.0), "beta1 and beta2"), (dict(beta2=-0.1), "beta1 and beta2"), (dict(beta1=float("nan")), "beta1 and beta2"),
    (dict(eps=0.0), "eps must be"), (dict(eps=float("nan")), "eps must be"), (dict(weight_decay=-1.0), "weight_decay must be"),
    (dict(count=-1), "count must be in"), (dict(tensors=None), "tensors is NULL"),
])
def test_refusals(lib, change, said):
    err = C.create_string_buffer(1024)
    a = _args(**change)
    assert lib.so3lr_adamw(C.byref(a), 256, 1 << 20, None, err, 1024) == 1
    assert said in err.value.decode(), err.value


def test_workspace(lib):
    err = C.create_string_buffer(1024)
    a = _args()
    need = lib.so3lr_adamw_workspace(C.byref(a))
    assert need > 0
    assert lib.so3lr_adamw(C.byref(a), 256, need - 1, None, err, 1024) == 1 and b"the workspace has" in err.value
    assert lib.so3lr_adamw(C.byref(a), 128, need, None, err, 1024) == 1 and b"workspace is not aligned" in err.value
    assert lib.so3lr_adamw(C.byref(a), None, need, None, err, 1024) == 1 and b"workspace is NULL" in err.value
    assert lib.so3lr_adamw_workspace(C.byref(_Adamw(-1))) == -1
    assert lib.so3lr_adamw(C.byref(_Adamw(0, None, 1e-3, None, 0.9, 0.999, 1e-8, 0.0)), None, 0, None, err, 1024) == 0
    assert lib.so3lr_adamw(None, None, 0, None, err, 1024) == 1 and b"args is NULL" in err.value


@pytest.mark.parametrize("change, said", [
    (dict(n=-1), "n must be in"), (dict(dtype=7), "dtype must be"), (dict(codes=None), "codes is NULL"),
    (dict(scales=2), "scales is not aligned"), (dict(values=None), "values is NULL"), (dict(values=3), "values is not aligned"),
])
def test_moment_values_refusals(lib, change, said):
    err = C.create_string_buffer(1024)
    a = _Values(10, 1, 1, 64, 128, 256)
    for k, v in change.items():
        setattr(a, k, v)
    assert lib.so3lr_moment_values(C.byref(a), None, err, 1024) == 1
    assert said in err.value.decode(), err.value


def test_optimizer_arguments():
    torch = pytest.importorskip("torch")
    optim = pytest.importorskip("so3lr_b200.optim")
    w = torch.nn.Parameter(torch.ones(3))
    with pytest.raises(ValueError, match="moment_bits must be 8 or 32"):
        optim.AdamW([w], moment_bits=4)
    with pytest.raises(ValueError, match="moment_bits must be 8 or 32"):
        optim.AdamW([dict(params=[w], moment_bits=16)])
    w.grad = torch.ones(3)
    with pytest.raises(ValueError, match="no CPU path"):
        optim.AdamW([w]).step()
