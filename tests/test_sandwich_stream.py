"""What sandwich_norm keeps of its arguments for its gradients (so3lr_b200.layers) on the GPU."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def layers():
    from so3lr_b200 import layers
    return layers


def _inputs(scale):
    g = torch.Generator(device="cuda").manual_seed(3)
    draw = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    x, residual, gate = (draw(33, 264).bfloat16() for _ in range(3))
    weight, following = (1 + 0.1 * draw(264) for _ in range(2))
    return [t.requires_grad_() for t in (x, residual, weight, following, gate)] + \
        [1 + 0.1 * draw(264) if scale else None], draw(33, 264).bfloat16()


def test_stream_without_scale_is_not_kept(layers):
    """Without a residual scale no gradient reads the residual: it may be written after the call, as its
    storage may be given back."""
    args, dy = _inputs(False)
    y, s = layers.sandwich_norm(*args)
    (y.float() * dy.float() + s.float()).sum().backward()
    want = [t.grad.clone() for t in args[:5]]
    again = [t.detach().clone().requires_grad_() for t in args[:5]]
    stream = again[1] * 1  # no leaf: a leaf that requires a gradient cannot be written
    y, s = layers.sandwich_norm(again[0], stream, *again[2:])
    with torch.no_grad():
        stream.zero_()
    (y.float() * dy.float() + s.float()).sum().backward()
    for a, b in zip(want, again):
        assert torch.equal(a, b.grad)


def test_stream_with_scale_is_kept(layers):
    """With one it is read, and a change of it is refused as torch refuses it."""
    args, dy = _inputs(True)
    stream = args[1] * 1
    y, s = layers.sandwich_norm(args[0], stream, *args[2:5], args[5].requires_grad_())
    with torch.no_grad():
        stream.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        (y.float() * dy.float() + s.float()).sum().backward()
