"""What the row-wise feed-forward layers do with derivatives that they do not compute."""
import pytest

torch = pytest.importorskip("torch")
from so3lr_b200.build import torch_module  # noqa: E402

if torch_module() is None:
    pytest.skip("the layers' module is not built here", allow_module_level=True)
import torch.autograd.forward_ad as fwd  # noqa: E402


@pytest.fixture(scope="module")
def layers():
    from so3lr_b200 import layers
    return layers


def _calls(layers, device):
    """Each call by name, as a function of its first floating tensor, and that tensor."""
    x, w = torch.randn(4, 64, device=device).bfloat16(), torch.ones(64, device=device)
    m = torch.randn(64, 64, device=device).bfloat16()
    c, one = torch.ones(4, 64, dtype=torch.int8, device=device), torch.ones(4, device=device)
    return {
        "rms_norm": (lambda t: layers.rms_norm(t, w), x),
        "rms_norm weight": (lambda t: layers.rms_norm(x, t), w),
        "rms_norm residual": (lambda t: layers.rms_norm(x, w, t), x),
        "rms_norm_int8": (lambda t: layers.rms_norm_int8(t, w), x),
        "rms_norm_backward": (lambda t: layers.rms_norm_backward(t, x, w), x),
        "feed_forward": (lambda t: layers.feed_forward(t, m, m, m), x),
        "feed_forward weight": (lambda t: layers.feed_forward(x, m, m, t), m),
        "feed_forward_train": (lambda t: layers.feed_forward_train(x, t, m, m), m),
        "gate_int8": (lambda t: layers.gate_int8(t), x),
        "int8_linear": (lambda t: layers.int8_linear(c, t, c, one), one),
        "int8_linear bias": (lambda t: layers.int8_linear(c, one, c, one, t), one),
        "dequantize_int8": (lambda t: layers.dequantize_int8(c, t), one),
    }


def test_forward_mode_is_refused(layers):
    """Also where the tensor is elsewhere than on a GPU: the tangent is looked at first."""
    for name, (call, t) in _calls(layers, "cpu").items():
        with fwd.dual_level():
            with pytest.raises(ValueError, match="forward-mode tangent|there is no CPU path|on cpu"):
                call(fwd.make_dual(t, torch.ones_like(t)))
    with fwd.dual_level(), pytest.raises(ValueError, match="x has a forward-mode tangent"):
        x = torch.zeros(4, 64, dtype=torch.bfloat16)
        layers.rms_norm(fwd.make_dual(x, x), torch.ones(64))


@pytest.mark.gpu
def test_forward_mode_is_refused_on_the_gpu(layers):
    for name, (call, t) in _calls(layers, "cuda").items():
        call(t)
        with fwd.dual_level():
            with pytest.raises(ValueError, match="forward-mode tangent"):
                call(fwd.make_dual(t, torch.ones_like(t)))
        with pytest.raises((ValueError, RuntimeError)):
            torch.func.jvp(call, (t,), (torch.ones_like(t),))
    # with a gradient in reverse mode as well, autograd itself refuses
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    with fwd.dual_level(), pytest.raises((ValueError, RuntimeError, NotImplementedError)):
        layers.rms_norm(fwd.make_dual(x, torch.ones_like(x)), torch.ones(64, device="cuda"))


def _traced(call, t):
    with pytest.raises(Exception, match="torch.jit.trace cannot record"), torch.no_grad():
        torch.jit.trace(call, (t,), check_trace=False)


def test_tracing_is_refused(layers):
    """A trace would hold the results of the traced call as constants."""
    x = torch.zeros(4, 64)
    _traced(lambda t: layers.rms_norm(t, torch.ones(64))[0], x)
    _traced(lambda t: layers.feed_forward(t, x, x, x), x)
    _traced(lambda t: layers.gate_int8(t)[1], x)


@pytest.mark.gpu
def test_tracing_is_refused_on_the_gpu(layers):
    for name, (call, t) in _calls(layers, "cuda").items():
        _traced(lambda v: torch.zeros(1, device="cuda") + (call(v) if torch.is_tensor(call(v)) else call(v)[1]).sum(), t)
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    with pytest.raises(Exception, match="torch.jit.trace cannot record"):
        torch.jit.trace(lambda t: layers.rms_norm(t, torch.ones(64, device="cuda"))[0], (x,), check_trace=False)
    layers.rms_norm(x, torch.ones(64, device="cuda"))


@pytest.mark.gpu
def test_eight_bit_calls_are_detached(layers):
    """The stream with a residual and without one alike, whatever requires a gradient."""
    x, r = (torch.randn(4, 64, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    w = torch.ones(64, device="cuda", requires_grad=True)
    for residual in (None, r, r.detach()):
        codes, scales, s = layers.rms_norm_int8(x, w, residual)
        assert not s.requires_grad and not scales.requires_grad
        if residual is None:
            assert s.data_ptr() == x.data_ptr() and torch.equal(s, x)
    assert layers.rms_norm_int8(r.detach(), w)[2] is not None
    plain = r.detach()
    assert layers.rms_norm_int8(plain, w)[2] is plain  # nothing to detach
    b, one = codes[:2], torch.ones(2, device="cuda", requires_grad=True)
    assert not layers.int8_linear(codes, scales, b, one, one).requires_grad
    assert not layers.dequantize_int8(codes, torch.ones(4, device="cuda", requires_grad=True)).requires_grad
    assert not layers.gate_int8(x)[1].requires_grad
    y, _ = layers.rms_norm(x, w, r)
    assert y.requires_grad
    with torch.no_grad():
        for residual in (None, r):
            assert not any(t.requires_grad for t in layers.rms_norm(x, w, residual))


@pytest.mark.gpu
def test_eps_that_is_no_number(layers):
    x, w = torch.zeros(2, 64, device="cuda"), torch.ones(64, device="cuda")
    for wrong in ("1e-6", None, [1e-6]):
        with pytest.raises(ValueError, match="eps must be a number"):
            layers.rms_norm(x, w, eps=wrong)
        with pytest.raises(ValueError, match="eps must be a number"):
            layers.rms_norm_backward(x, x, w, eps=wrong)
    layers.rms_norm(x, w, eps=torch.tensor(1e-6))
