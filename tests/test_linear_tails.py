"""The tail of gelu (so3lr_b200.layers.linear), where z Phi(z) is far below z, on the GPU against
float64.

u is a type's unit roundoff (2^-8 bfloat16, 2^-11 float16), U = 2^-24. x is z: the weight is 1. Phi(-|z|) is
t poly(t) exp(-z^2 / 2), the polynomial within 6e-6 of it relative to its value. The exponent is two
rounded products and a rounded constant, 3 U (z^2 / 2) of the result; the hardware's reciprocal and
exponential, the polynomial's and the last products' roundings are 20 U. At |z| <= 12 that is 1.3e-5 + 6e-6 +
1.2e-6 = 2.0e-5, below 2^-15; for positive z, 1 - Phi(-|z|) adds a rounding. y is then rounded to its type.
The slope is Phi(z) + z phi(z), each part within 2^-15 of itself; a float32 bias gradient of one row is the slope
itself, rounded with its sum (2 U)."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U32, FUN = 2.0 ** -24, 2.0 ** -15
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


@pytest.fixture(scope="module")
def layers():
    from so3lr_b200 import layers
    return layers


def _parts(z):
    """Phi(z) and z phi(z) in float64"""
    return 0.5 * torch.erfc(-z / math.sqrt(2)), z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def _within(got, want, bound, what):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    at = bad.nonzero()[0].tolist() if bool(bad.any()) else None
    assert at is None, f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, first at {at}: {off[bad][0]:.3e} > {bound[bad][0]:.3e}"


@pytest.mark.parametrize("dtype", list(U))
def test_gelu_tail(layers, dtype):
    x = torch.linspace(-12, 12, 4001, dtype=torch.float64, device="cuda").to(dtype)[:, None]
    w = torch.ones(1, 1, device="cuda", dtype=dtype)
    for rows in (x, *x[:1300].split(13)[:40], x[1500:1513]):  # many rows, and few
        y, saved = layers.linear_train(rows, w, activation="gelu")
        z = rows.double()
        cdf, rise = _parts(z)
        want = z * cdf
        _within(y, want, (U[dtype] + FUN * (1 + U[dtype])) * want.abs() + TINY[dtype], "y")
        dx, _, _ = layers.linear_backward(torch.ones_like(y), saved)
        slope, size = cdf + rise, cdf + rise.abs()
        _within(dx, slope, U[dtype] * slope.abs() + (1 + U[dtype]) * FUN * size + TINY[dtype], "slope")


def test_gelu_tail_in_split_contractions(layers):
    """A contraction that is cut into parts: each activation is formed where the parts are joined."""
    k, dtype = 16384, torch.bfloat16
    z = torch.linspace(-12, 12, 256, dtype=torch.float64, device="cuda").to(dtype)
    x = torch.zeros(256, k, device="cuda", dtype=dtype)
    x[torch.arange(256), torch.arange(256) * 64 + 1] = z
    w = torch.ones(8, k, device="cuda", dtype=dtype)
    y = layers.linear(x, w, activation="gelu")
    want = (z.double() * _parts(z.double())[0])[:, None].expand(256, 8)
    _within(y, want, (U[dtype] + FUN * (1 + U[dtype])) * want.abs() + TINY[dtype], "y")


@pytest.mark.parametrize("dtype", list(U))
def test_gelu_slope_in_32_bits(layers, dtype):
    """One row, channels with a z of their own: the float32 bias gradient is the slope."""
    z = torch.linspace(-12, 12, 4001, dtype=torch.float64, device="cuda").to(dtype)
    bias = torch.zeros(4001, device="cuda")
    x = torch.ones(1, 1, device="cuda", dtype=dtype)
    y, saved = layers.linear_train(x, z[:, None].contiguous(), bias, activation="gelu")
    _, _, db = layers.linear_backward(torch.ones_like(y), saved)
    cdf, rise = _parts(z.double())
    assert db.dtype == torch.float32
    _within(db, cdf + rise, FUN * (cdf + rise.abs()) + 2 * U32 * (cdf + rise).abs(), "slope")
