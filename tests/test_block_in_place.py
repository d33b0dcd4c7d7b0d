"""Results of the dense layer and of the norms on both sides of a block in the memory of their
inputs, which the C entry points allow (the Python calls allocate theirs), and their waits
when they run out."""
import ctypes as C
import pathlib
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_block_abi import _Linear, _Sandwich  # noqa: E402

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


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


def _rand(seed, *shape, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows, width", [(1, 1), (9, 40), (300, 96), (77, 256), (50, 515), (33, 1003), (4000, 1536), (3000, 2048),
                                         (3, 8187), (2, 16384)])
def test_sandwich_norm_in_place(layers, rows, width, dtype):
    x, r, g = (_rand(i, rows, width, dtype=dtype) for i in (1, 2, 3))
    w, n, c = (_rand(i, width, dtype=dtype) for i in (4, 5, 6))
    want_y, want_s = layers.sandwich_norm(x, r, w, n, g, c)
    for s_in, y_in in (("x", "residual"), ("residual", "gate"), ("gate", "x"), ("x", None), (None, "x")):
        own = dict(x=x.clone(), residual=r.clone(), gate=g.clone())
        a = _Sandwich(rows=rows, width=width, dtype=TYPES[dtype], weight_dtype=TYPES[dtype], eps=1e-6, weight=w.data_ptr(),
                      next_weight=n.data_ptr(), residual_scale=c.data_ptr())
        s = own[s_in] if s_in else torch.empty_like(x)
        y = own[y_in] if y_in else torch.empty_like(x)
        for k, v in dict(own, s=s, y=y).items():
            setattr(a, k, v.data_ptr())
            setattr(a, k + "_stride", width)
        _call("so3lr_sandwich_norm", a)
        assert torch.equal(s, want_s) and torch.equal(y, want_y), (s_in, y_in)


@pytest.mark.parametrize("rows, k, n", [(3, 64, 96), (16, 250, 131), (300, 256, 512), (333, 100, 251), (300, 20000, 256)])
def test_linear_in_place(layers, rows, k, n):
    """y in the residual's memory: few rows, whole tiles, rows off the boundaries, split contractions."""
    from so3lr_b200 import load_library
    dtype = torch.bfloat16
    x, w, r = _rand(1, rows, k, dtype=dtype), _rand(2, n, k, dtype=dtype) * k ** -0.5, _rand(3, rows, n, dtype=dtype)
    b = _rand(4, n, dtype=torch.float32)
    want = layers.linear(x, w, b, r, activation="gelu")
    y = r.clone()
    a = _Linear(rows=rows, n=n, k=k, dtype=1, bias_dtype=0, activation=2, x=x.data_ptr(), x_stride=k, w=w.data_ptr(), w_stride=k,
                bias=b.data_ptr(), residual=y.data_ptr(), residual_stride=n, y=y.data_ptr(), y_stride=n)
    size = load_library().so3lr_linear_workspace
    size.restype = C.c_longlong
    need = size(C.byref(a))
    scratch = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    _call("so3lr_linear", a, C.c_void_p(scratch.data_ptr()), C.c_longlong(need))
    assert torch.equal(y, want)


def _until_it_gives_up(layers, call, limits, stages):
    """Runs `call` with short limits: it ends, the host hears of it, and the next calls are right."""
    from so3lr_b200 import So3lrError
    want, gave_up = call(), 0
    try:
        for limit in limits:
            layers.set_wait_limit(limit)
            for _ in range(2):
                try:
                    got = call()
                    torch.cuda.synchronize()
                    layers.check_status()
                    assert all(torch.equal(a, b) for a, b in zip(got, want))  # no wait was too long
                except So3lrError as e:
                    assert any(f"gave up waiting (stage {s})" in str(e) for s in stages), e
                    gave_up += 1
                    torch.cuda.synchronize()  # a call of the step was refused: the one before it has ended
                    try:
                        layers.check_status()
                    except So3lrError:
                        pass
            layers.set_wait_limit()
            assert all(torch.equal(a, b) for a, b in zip(call(), want))
    finally:
        layers.set_wait_limit()
    assert gave_up >= 1


@pytest.mark.parametrize("rows, width", [(6000, 1024), (2600, 4096), (2400, 8192)])
def test_sandwich_rings_end_when_a_wait_runs_out(layers, rows, width):
    x, r, g, dy, ds = (_rand(i, rows, width, dtype=torch.bfloat16) for i in range(5))
    w = torch.ones(width, device="cuda")
    s = layers.sandwich_norm(x, r, w, w, g, w)[1]
    for call in (lambda: layers.sandwich_norm(x, r, w, w, g, w), lambda: layers.sandwich_norm(x, r, w, w),
                 lambda: layers.sandwich_norm_backward(dy, ds, s, x, r, w, w, g, w),
                 lambda: layers.sandwich_norm_backward(dy, None, s, x, r, w, w)[:4]):
        _until_it_gives_up(layers, call, (1, 300, 700, 1500, 3000), (7,))


@pytest.mark.parametrize("rows, k, n", [(3000, 256, 1024), (700, 1032, 1368), (300, 91, 251), (600, 16384, 256)])
def test_linear_ends_when_a_wait_runs_out(layers, rows, k, n):
    x, w, r = _rand(1, rows, k, dtype=torch.bfloat16), _rand(2, n, k, dtype=torch.bfloat16) * k ** -0.5, _rand(3, rows, n, dtype=torch.bfloat16)
    b, dy = _rand(4, n, dtype=torch.float32), _rand(5, rows, n, dtype=torch.bfloat16)
    for call in (lambda: (layers.linear(x, w, b, r, activation="silu"),),
                 lambda: layers.linear_backward(dy, layers.linear_train(x, w, b, r, activation="silu")[1])):
        _until_it_gives_up(layers, call, (1, 500, 1500, 4000, 15000), range(1, 7))


@pytest.mark.parametrize("call", ["layers.linear(x, m, w, x, activation='gelu')", "layers.linear(big, m, w, big)",
                                  "layers.sandwich_norm(x, x, w, w)", "layers.sandwich_norm(big, big, w, w)",
                                  "optim.moment_values(c, w)"])
def test_the_first_call_of_a_process_may_be_captured(call):
    program = f"""
import torch
from so3lr_b200 import layers, optim
x, big, m = (torch.randn(n, 1024, device="cuda").bfloat16() for n in (10, 6000, 1024))
w, c = torch.randn(1024, device="cuda"), torch.ones(1024, 256, dtype=torch.int8, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = {call}
graph.replay()
torch.cuda.synchronize()
want = {call}
pairs = zip(got, want) if isinstance(got, tuple) else [(got, want)]
assert all(torch.equal(a, b) for a, b in pairs)
layers.check_status()
print("captured")
"""
    root = pathlib.Path(__file__).resolve().parents[1]
    res = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=120, cwd=root)
    assert res.returncode == 0 and "captured" in res.stdout, res.stdout + res.stderr
