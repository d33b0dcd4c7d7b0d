"""Bounded waits of the row-wise feed-forward kernels: what a call says when a wait of
an earlier one has given up."""
import ctypes as C
import pathlib
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def layers():
    from so3lr_b200 import layers
    return layers


def _calls(layers):
    """One call of each kind that queues work: dense and few-row products, row kernels with and without a ring."""
    half = lambda *n: torch.randn(*n, device="cuda").bfloat16()  # noqa: E731
    ones = lambda n: torch.ones(n, device="cuda")  # noqa: E731
    x, w, d = half(300, 64), half(96, 64), half(64, 96)
    big = half(6000, 1024)
    _, saved = layers.feed_forward_train(x, w, w, d)
    c = torch.ones(300, 64, dtype=torch.int8, device="cuda")
    return {
        "feed_forward": lambda: layers.feed_forward(x, w, w, d),
        "feed_forward, few rows": lambda: layers.feed_forward(x[:2], w, w, d),
        "feed_forward_backward": lambda: layers.feed_forward_backward(x, saved),
        "int8_linear": lambda: layers.int8_linear(c, ones(300), c, ones(300)),
        "int8_linear, few rows": lambda: layers.int8_linear(c[:2], ones(2), c, ones(300)),
        "rms_norm": lambda: layers.rms_norm(x, ones(64)),
        "rms_norm_backward": lambda: layers.rms_norm_backward(x, x, ones(64)),
        "rms_norm_backward, ring": lambda: layers.rms_norm_backward(big, big, ones(1024)),
        "rms_norm_int8": lambda: layers.rms_norm_int8(x, ones(64)),
        "rms_norm_int8, ring": lambda: layers.rms_norm_int8(big, ones(1024)),
        "gate_int8": lambda: layers.gate_int8(x),
        "dequantize_int8": lambda: layers.dequantize_int8(c, ones(300)),
    }


def test_a_wait_that_gave_up_is_reported_once(layers):
    """The word that a kernel writes, written here by the host: every kind of call is refused until
    check_status has said so, and accepted afterwards."""
    from so3lr_b200 import So3lrError, load_library
    word = getattr(load_library(), "_ZN10so3lr_b20012gave_up_flagEv")
    word.restype = C.POINTER(C.c_int)
    calls = _calls(layers)
    layers.check_status()
    for name, call in calls.items():
        call()
        torch.cuda.synchronize()
        word()[0] = 3
        for _ in range(2):
            with pytest.raises(So3lrError, match="gave up waiting .stage 3.*so3lr_layers_status"):
                call()
        with pytest.raises(So3lrError, match="gave up waiting .stage 3"):
            layers.check_status("cuda:0")
        layers.check_status()
        call()
    torch.cuda.synchronize()
    layers.check_status(torch.device("cuda"))
    # what queues nothing is not refused, and takes nothing from the report
    word()[0] = 5
    assert layers.rms_norm(torch.zeros(0, 64, device="cuda"), torch.ones(64, device="cuda"))[0].shape == (0, 64)
    with pytest.raises(So3lrError, match="stage 5"):
        layers.check_status()


def _rows(rows, width, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    return [torch.randn(rows, width, generator=g, device="cuda").to(dtype) for _ in range(3)]


@pytest.mark.parametrize("rows, width", [(6000, 1024), (2600, 4096), (2400, 8192), (5003, 1536)])
def test_ring_kernels_end_when_a_wait_runs_out(layers, rows, width):
    """Rows come from HBM in about 1,500 cycles: with shorter limits blocks give up at their first rows
    or later ones, with their copies in flight. The kernel ends, the host hears of it, and the next
    calls are right, in the same memory."""
    from so3lr_b200 import So3lrError
    x, r, dy = _rows(rows, width, torch.bfloat16)
    w = torch.ones(width, device="cuda")
    calls = (lambda: layers.rms_norm_int8(x, w), lambda: layers.rms_norm_int8(x, w, r),
             lambda: layers.rms_norm_backward(dy, x, w), lambda: layers.rms_norm_backward(dy, x, w, r))
    for call in calls:
        want = call()
        gave_up = 0
        try:
            for limit in (1, 300, 700, 1500, 3000):
                layers.set_wait_limit(limit)
                got = call()
                torch.cuda.synchronize()
                try:
                    layers.check_status()
                    assert all(torch.equal(a, b) for a, b in zip(got, want))  # no wait was too long
                except So3lrError as e:
                    assert "stage 7" in str(e)
                    gave_up += 1
                layers.set_wait_limit()
                assert all(torch.equal(a, b) for a, b in zip(call(), want))
        finally:
            layers.set_wait_limit()
        assert gave_up >= 1


def _product(layers, kind):
    g = torch.Generator(device="cuda").manual_seed(5)
    half = lambda *n: torch.randn(*n, generator=g, device="cuda").mul_(n[-1] ** -0.5).bfloat16()  # noqa: E731
    if kind.startswith("int8"):
        rows, n, k = {"int8 ragged": (333, 1531, 1000), "int8 split": (600, 256, 16384), "int8 waves": (3000, 4096, 512)}[kind]
        a, b = (torch.randint(-127, 128, s, generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
                for s in ((rows, k), (n, k)))
        sa, sb = torch.rand(rows, device="cuda"), torch.rand(n, device="cuda")
        return lambda: (layers.int8_linear(a, sa, b, sb),)
    rows, width, hidden = {"narrow": (3000, 256, 1024), "wide": (700, 1032, 1368), "unaligned": (300, 91, 251)}[kind]
    x, dy, wg, wu, wd = half(rows, width), half(rows, width), half(hidden, width), half(hidden, width), half(width, hidden)

    def step():
        y, saved = layers.feed_forward_train(x, wg, wu, wd)
        return (y, *layers.feed_forward_backward(dy, saved))
    return step


@pytest.mark.parametrize("kind", ["int8 ragged", "int8 split", "int8 waves", "narrow", "wide", "unaligned"])
def test_products_end_when_a_wait_runs_out(layers, kind):
    """The first K block takes about 1,500 cycles to come, a tile's accumulator some thousands: with
    these limits CTA pairs give up at loads, products or epilogues, with copies and products in flight,
    one CTA before the other. The kernels end, the host hears of it, and the next calls are right."""
    from so3lr_b200 import So3lrError
    step = _product(layers, kind)
    want = step()
    gave_up = 0
    try:
        for limit in (1, 200, 500, 1000, 1500, 2000, 3000, 5000, 8000, 15000):
            layers.set_wait_limit(limit)
            for _ in range(3):
                try:
                    got = step()
                    torch.cuda.synchronize()
                    layers.check_status()
                    assert all(torch.equal(a, b) for a, b in zip(got, want))  # no wait was too long
                except So3lrError as e:
                    assert "gave up waiting (stage " in str(e) and 1 <= int(str(e).split("stage ")[1][0]) <= 6
                    gave_up += 1
                    torch.cuda.synchronize()  # a call of the step was refused: the one before it has ended
                    try:
                        layers.check_status()
                    except So3lrError:
                        pass
            layers.set_wait_limit()
            assert all(torch.equal(a, b) for a, b in zip(step(), want))
    finally:
        layers.set_wait_limit()
    assert gave_up >= 1


def test_the_limit_is_a_waits_and_not_a_kernels(layers):
    """Products of 0.8 ms and more under a limit of 0.2 ms: a tile takes 10 to 40 us, and every wait is for one
    step of the pipeline."""
    g = torch.Generator(device="cuda").manual_seed(7)
    a, b = (torch.randint(-127, 128, s, generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
            for s in ((32768, 4096), (8192, 4096)))
    sa, sb = torch.rand(32768, device="cuda"), torch.rand(8192, device="cuda")
    x, wg, wu, wd = (torch.randn(*s, generator=g, device="cuda").mul_(s[-1] ** -0.5).bfloat16()
                     for s in ((65536, 1024), (4096, 1024), (4096, 1024), (1024, 4096)))
    for call in (lambda: layers.int8_linear(a, sa, b, sb), lambda: layers.feed_forward(x, wg, wu, wd)):
        want = call()
        torch.cuda.synchronize()
        try:
            layers.set_wait_limit(400_000)
            got = call()
            torch.cuda.synchronize()
            layers.check_status()
        finally:
            layers.set_wait_limit()
        assert torch.equal(got, want)


@pytest.mark.parametrize("call", ["layers.rms_norm(x, w)", "layers.rms_norm_int8(big, w)", "layers.gate_int8(x)",
                                  "layers.feed_forward(x[:2], m, m, m)", "layers.feed_forward(big, m, m, m)",
                                  "layers.int8_linear(c, s, c, s)"])
def test_the_first_call_of_a_process_may_be_captured(call):
    """It makes the words that waits which give up are reported in, and sets up kernels and tensor maps."""
    program = f"""
import torch
from so3lr_b200 import layers
x, big, m, w = (torch.randn(n, 1024, device="cuda").bfloat16() for n in (40, 6000, 1024, 1))
w, c, s = w[0].float(), torch.ones(300, 64, dtype=torch.int8, device="cuda"), torch.ones(300, device="cuda")
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
