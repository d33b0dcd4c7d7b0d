"""Weight decay far below float32's spacing at 1 (so3lr_b200.optim) on the GPU, against the
formula in float64.

u is 2^-24. Without gradients and moments a step is p - lr weight_decay p, which is rounded
once: the product lr weight_decay is within 2 u of itself (lr on the GPU is a float32, and the
product is rounded to one). 1 - lr weight_decay is two floats, the second of at most 2^-22 and
rounded, 2^-47 at most, as is its product with p, 2^-46 |p| at most: p is off by half its unit, 4 u
of the decay and 2^-45 |p|. With gradients the update adds its own errors, 32 u of
lr / bc1 |m| / (sqrt(v / bc2) + eps), as the tests of whole steps have it, and what is added to p is
rounded once more: u of it.
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U32 = 2.0 ** -24
N = 4096 + 77


@pytest.fixture(scope="module")
def optim():
    from so3lr_b200 import optim
    return optim


def _half_unit(p):
    return torch.ldexp(torch.ones_like(p), torch.frexp(p).exponent - 25)


@pytest.mark.parametrize("on_gpu", [False, True])
@pytest.mark.parametrize("kind", ["float32", "master", "eight"])
@pytest.mark.parametrize("lr, decay", [(1e-5, 1e-2), (2e-5, 1e-2), (2e-6, 1e-2), (3e-4, 0.1), (0.5, 1.0)])
@pytest.mark.parametrize("gradients", [False, True])
def test_small_decay(optim, lr, decay, kind, on_gpu, gradients):
    g = torch.Generator(device="cuda").manual_seed(1)
    p = torch.randn(N, generator=g, device="cuda")
    grad = torch.randn(N, generator=g, device="cuda") * 1e-2 if gradients else torch.zeros(N, device="cuda")
    dtype = torch.bfloat16 if kind == "master" else torch.float32
    param, master = p.to(dtype, copy=True), p.clone() if kind == "master" else None
    if kind == "eight":
        blocks = (N + 255) // 256
        m, v = torch.zeros(N, dtype=torch.int8, device="cuda"), torch.zeros(N, dtype=torch.uint8, device="cuda")
        scales = [torch.zeros(blocks, device="cuda")], [torch.zeros(blocks, device="cuda")]
    else:
        m, v = torch.zeros(N, device="cuda"), torch.zeros(N, device="cuda")
        scales = None, None
    rate = torch.tensor(lr, device="cuda") if on_gpu else lr
    optim.adamw_step([param], [grad], [m], [v], torch.zeros(1, dtype=torch.int64, device="cuda"),
                     exp_avg_scales=scales[0], exp_avg_sq_scales=scales[1], masters=None if master is None else [master],
                     lr=rate, betas=(0.9, 0.999), eps=1e-8, weight_decay=decay)
    got = (param if master is None else master).double()
    p, grad = p.double(), grad.double()
    m1, v1 = 0.1 * grad, 1e-3 * grad * grad
    update = lr / (1 - 0.9) * m1 / ((v1 / (1 - 0.999)).sqrt() + 1e-8)
    want = p - lr * decay * p - update
    slack = (4 * U32 * lr * decay + 2.0 ** -45) * p.abs() + 33 * U32 * (update.abs() + lr * decay * p.abs()) * float(gradients)
    half = torch.maximum(_half_unit(p), _half_unit(want))
    off = (got - want).abs()
    bad = off > half + slack
    assert not bool(bad.any()), (f"{int(bad.sum())} of {N}, the worst by {float((off / half).max()):.3f} half units; "
                                 f"mean of the change / decay {float(((got - p + update) / p).mean() / -(lr * decay)):.4f}")


@pytest.mark.parametrize("lr, decay", [(1e-5, 0.0), (1e-5, 1e-2), (1e-5, 0.1), (1e-5, 1.0), (0.5, 1.0), (0.25, 2.0)])
def test_infinite_parameters_stay(optim, lr, decay):
    """A parameter of minus infinity, as a mask has them, is decayed to itself; a NaN stays one."""
    p = torch.linspace(-1, 1, 300, device="cuda")
    p[::7], p[1::7], p[2::7] = -float("inf"), float("inf"), float("nan")
    got, zeros = p.clone(), lambda: torch.zeros_like(p)  # noqa: E731
    optim.adamw_step([got], [zeros()], [zeros()], [zeros()], torch.zeros(1, dtype=torch.int64, device="cuda"), lr=lr,
                     weight_decay=decay)
    assert torch.equal(got.isnan(), p.isnan())
    assert torch.equal(got[p.isinf()], p[p.isinf()]) and bool(got[p.isfinite()].isfinite().all())
    if decay == 0.0:
        assert torch.equal(got[p.isfinite()], p[p.isfinite()])
