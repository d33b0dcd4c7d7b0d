"""8-bit rows whose values are near the bottom of float32's range."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F32 = 64 * 2.0 ** -24  # as in test_layers.py


@pytest.fixture(scope="module")
def layers():
    from so3lr_b200 import layers
    return layers


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, width", [(5, 60), (7, 100), (300, 256), (4, 1003), (3, 2048), (6000, 1536), (2, 16384)])
def test_rms_norm_int8_of_tiny_products(layers, rows, width, dtype):
    """max|s w| down to 2^-124, below which 127 / max|s w| is no float32: the row's root mean square is below
    sqrt(eps), so y is a thousand times larger and its scale an ordinary number. Codes are exact: no value is
    near the middle between two."""
    part = torch.tensor([1.0, 0.0, -1.0, 0.25, -0.75, 0.0, 0.6], device="cuda", dtype=torch.float64)
    want = torch.tensor([127, 0, -127, 32, -95, 0, 76], device="cuda", dtype=torch.int8)
    which = torch.arange(rows * width, device="cuda").view(rows, width) * 5 % 7
    want = want[which]
    sizes = 2.0 ** -torch.tensor([100, 101, 114, 119, 121, 122, 124], device="cuda", dtype=torch.float64)
    size = sizes[torch.arange(rows, device="cuda") % 7][:, None]
    # float16 has no such numbers: the weight is as small instead
    lift = 2.0 ** 110 if dtype is torch.float16 else 1.0
    x = (part[which] * size * lift).to(dtype)
    w = torch.full((width,), 1 / lift, device="cuda")
    codes, scales, s = layers.rms_norm_int8(x, w, eps=1e-6)
    y = s.double() * w.double() * (s.double().square().mean(1, keepdim=True) + 1e-6).rsqrt()
    scale = y.abs().amax(1) / 127
    assert bool((scale > 2.0 ** -126).all())
    assert bool(((scales.double() - scale).abs() <= F32 * scale).all())
    assert torch.equal(codes, want)
