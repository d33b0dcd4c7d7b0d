"""Results of the row kernels in the memory of their inputs, which the C entry points allow
(the Python calls allocate theirs): the same bits as with memory of their own."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
import ctypes as C  # noqa: E402

from test_layers_abi import _RmsNorm, _RmsNormBackward  # noqa: E402

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
SIZES = [(1, 1), (9, 40), (300, 96), (77, 256), (50, 515), (33, 1003), (6000, 1536), (3000, 2048), (3, 8187), (2, 16384)]


@pytest.fixture(scope="module")
def layers():
    from so3lr_b200 import layers
    return layers


def _call(name, args, *workspace):
    from so3lr_b200 import load_library
    err = C.create_string_buffer(512)
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    rc = getattr(load_library(), name)(C.byref(args), *workspace, stream, err, C.c_size_t(512))
    assert rc == 0, err.value


def _rows(seed, rows, width, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(rows, width, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows, width", SIZES)
def test_norm_in_place(layers, rows, width, dtype):
    w = torch.rand(width, device="cuda") + 0.5
    x0, r0 = _rows(1, rows, width, dtype), _rows(2, rows, width, dtype)
    want_y, want_s = layers.rms_norm(x0, w, r0)
    want_codes, want_scales, _ = layers.rms_norm_int8(x0, w, r0)

    def args(x, r, **kw):
        a = _RmsNorm(rows=rows, width=width, dtype=TYPES[dtype], weight_dtype=0, eps=1e-6, x=x.data_ptr(), x_stride=width,
                     weight=w.data_ptr())
        if r is not None:
            a.residual, a.residual_stride = r.data_ptr(), width
        for k, v in kw.items():
            setattr(a, k, v.data_ptr())
            if k != "scales":
                setattr(a, k + "_stride", v.stride(0))
        return a

    for s_is_x in (True, False):
        x, r = x0.clone(), r0.clone()
        s, y = (x, r) if s_is_x else (r, x)
        _call("so3lr_rms_norm", args(x, r, s=s, y=y))
        assert torch.equal(s, want_s) and torch.equal(y, want_y)
        x, r = x0.clone(), r0.clone()
        s = x if s_is_x else r
        codes, scales = torch.empty_like(want_codes.contiguous()), torch.empty_like(want_scales)
        _call("so3lr_rms_norm", args(x, r, s=s, codes=codes, scales=scales))
        assert torch.equal(s, want_s) and torch.equal(codes, want_codes) and torch.equal(scales, want_scales)
    x = x0.clone()
    _call("so3lr_rms_norm", args(x, None, y=x))
    assert torch.equal(x, layers.rms_norm(x0, w)[0])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows, width", SIZES)
def test_gradient_in_place(layers, rows, width, dtype):
    w = torch.rand(width, device="cuda") + 0.5
    s, dy0, ds0 = (_rows(k, rows, width, dtype) for k in (1, 2, 3))
    from so3lr_b200 import load_library
    size = load_library().so3lr_rms_norm_backward_workspace
    size.restype = C.c_longlong
    for with_ds in (True, False):
        want, want_dw = layers.rms_norm_backward(dy0, s, w, ds0 if with_ds else None)
        for into in ("dy", "ds") if with_ds else ("dy",):
            dy, ds = dy0.clone(), ds0.clone()
            dx = dy if into == "dy" else ds
            dw = torch.empty_like(w)
            a = _RmsNormBackward(rows=rows, width=width, dtype=TYPES[dtype], weight_dtype=0, eps=1e-6, dy=dy.data_ptr(),
                                 dy_stride=width, s=s.data_ptr(), s_stride=width, weight=w.data_ptr(), dx=dx.data_ptr(),
                                 dx_stride=width, dweight=dw.data_ptr())
            if with_ds:
                a.ds, a.ds_stride = ds.data_ptr(), width
            need = size(C.byref(a))
            scratch = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
            _call("so3lr_rms_norm_backward", a, C.c_void_p(scratch.data_ptr()), C.c_longlong(need))
            assert torch.equal(dx, want) and torch.equal(dw, want_dw)
