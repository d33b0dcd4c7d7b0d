"""The dense layer, the norms on both sides of a block and AdamW past 2^31 elements: the far
ends against float64 formulas. Bounds as in test_linear.py, test_sandwich_norm.py and
test_optim.py, whose checks are used."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_linear import ACC, FUN, U, _act  # noqa: E402
from test_optim import HYPER, _check  # noqa: E402
from test_sandwich_norm import F32, TINY, U32, _check_forward, _gradients, _within  # noqa: E402


@pytest.fixture(scope="module", autouse=True)
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 70 << 30:
        pytest.skip("needs 70 GB of device memory")
    yield
    torch.cuda.empty_cache()


def _rand(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for part in flat.split(1 << 27):
        part.copy_(torch.randn(part.numel(), generator=g, device="cuda").mul_(scale))
    return out


def test_linear():
    from so3lr_b200 import layers
    rows, k, n = 70001, 64, 32768
    x, w, b = _rand(1, rows, k), _rand(2, n, k, scale=0.125), _rand(3, n, dtype=torch.float32)
    dy = _rand(4, rows, n)
    assert dy.numel() > 1 << 31
    y, saved = layers.linear_train(x, w, b, dy, activation="silu")
    dx, dw, db = layers.linear_backward(dy, saved)
    u = U[torch.bfloat16]
    ends = torch.tensor([0, 1, 65535, 65537, rows - 2, rows - 1], device="cuda")
    z = x[ends].double() @ w.double().t() + b.double()
    err = (k + 1) * ACC * (x[ends].double().abs() @ w.double().abs().t() + b.double().abs())
    value, slope = _act(z, "silu")
    r = dy[ends].double()
    _within(y[ends], value + r, u * (value + r).abs() + (1 + u) * (1.2 * err + FUN * (1 + z.abs()) + U32 * (value.abs() + r.abs()))
            + 2.0 ** -133, "y")
    loose = r.abs() * (1.2 * (u + err) + FUN * (1 + z.abs()))
    dz, size = r * slope, r.abs() * slope.abs() * (1 + u) + loose * (1 + u)
    ref, wide = dz @ w.double(), size @ w.double().abs()
    _within(dx[ends], ref, u * ref.abs() + (1 + u) * ((loose * (1 + u) + u * dz.abs()) @ w.double().abs() + n * ACC * wide), "dx")
    for c in (0, 17, n - 1):  # a channel's gradients over all rows
        z = x.double() @ w[c].double() + b[c].double()
        _, slope = _act(z, "silu")
        d = dy[:, c].double()
        dz, loose = d * slope, d.abs() * (1.2 * (u + 1e-4) + FUN * (1 + z.abs()))
        assert abs(float(db[c]) - float(dz.sum())) <= float(loose.sum()) + rows * U32 * float(dz.abs().sum())
        ref = dz @ x.double()
        bound = u * ref.abs() + ((loose + u * dz.abs()) @ x.double().abs()) + rows * ACC * (dz.abs() @ x.double().abs())
        _within(dw[c], ref, bound, "dw")


def test_sandwich_norm():
    from so3lr_b200 import layers
    width = 1000
    rows = (1 << 31) // width + 5003
    t = dict(x=_rand(1, rows, width), residual=_rand(2, rows, width), gate=_rand(3, rows, width),
             weight=_rand(4, width), next_weight=_rand(5, width), residual_scale=_rand(6, width))
    assert t["x"].numel() > 1 << 31
    y, s = layers.sandwich_norm(**t)
    ends = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device="cuda")
    part = {k: v[ends] if v.dim() == 2 else v for k, v in t.items()}
    _check_forward(y[ends], s[ends], part)
    dy, ds = y, t["residual"]  # any rows of the shape
    out = layers.sandwich_norm_backward(dy, ds, s, **t)
    want = _gradients(part, s[ends], dy[ends], ds[ends])
    u = U[torch.bfloat16]
    for i, name in ((0, "dx"), (1, "dresidual"), (4, "dgate")):
        ref, size = want[name]
        _within(out[i][ends], ref, u * ref.abs() + 2 * F32 * size + TINY[torch.bfloat16], name)
    sums = {}
    for a in range(0, rows, 100000):
        rows_of = lambda v: v[a:a + 100000]  # noqa: E731
        got = _gradients({k: rows_of(v) if v.dim() == 2 else v for k, v in t.items()}, rows_of(s), rows_of(dy), rows_of(ds))
        for name in ("dweight", "dnext_weight", "dresidual_scale"):
            old = sums.get(name, (0.0, 0.0))
            sums[name] = old[0] + got[name][0], old[1] + got[name][1]
    for i, name in ((2, "dweight"), (3, "dnext_weight"), (5, "dresidual_scale")):
        ref, size = sums[name]
        # a block adds 1/148 of the rows or fewer one after the other
        _within(out[i], ref, u * ref.abs() + (rows / 148 * U32 + 2 * F32) * size + TINY[torch.bfloat16], name)


@pytest.mark.parametrize("eight", [False, True])
def test_adamw(eight):
    from so3lr_b200 import optim
    n = (1 << 31) + 2048 * 3 + 77
    g = torch.Generator(device="cuda").manual_seed(1)
    s = dict(p=[_rand(1, n)], g=[_rand(2, n, scale=0.01)], master=[None], ms=[None], vs=[None],
             steps=torch.tensor([7], device="cuda"))
    blocks = (n + 255) // 256
    if eight:
        s["m"] = [torch.randint(-127, 128, (n,), generator=g, device="cuda", dtype=torch.int8)]
        s["v"] = [torch.randint(1, 256, (n,), generator=g, device="cuda", dtype=torch.uint8)]
        s["ms"], s["vs"] = ([torch.rand(blocks, generator=g, device="cuda") * k + k] for k in (1e-3, 1e-5))
    else:
        s["m"], s["v"] = [_rand(3, n, dtype=torch.float32, scale=1e-3)], [_rand(4, n, dtype=torch.float32).abs_().mul_(1e-4)]
    spans = [(0, 1024), ((1 << 31) - 1024, (1 << 31) + 1024), (n // 256 * 256 - 2048, n)]

    def cut(k, a, b):
        v = s[k][0]
        return [None] if v is None else [v[a // 256:(b + 255) // 256].clone() if k in ("ms", "vs") else v[a:b].clone()]

    take = lambda a, b: {**{k: cut(k, a, b) for k in ("p", "g", "m", "v", "ms", "vs", "master")}, "steps": s["steps"].clone()}  # noqa: E731
    before = [take(a, b) for a, b in spans]
    optim.adamw_step(s["p"], s["g"], s["m"], s["v"], s["steps"], exp_avg_scales=s["ms"], exp_avg_sq_scales=s["vs"], **HYPER)
    for (a, b), old in zip(spans, before):
        _check(old, take(a, b), what=f"{a}..{b}")
    if eight:
        values = optim.moment_values(s["m"][0], s["ms"][0], torch.bfloat16)
        tail = optim.moment_values(s["m"][0][-77 - 256 * 3:].clone(), s["ms"][0][-4:].clone(), torch.bfloat16)
        assert torch.equal(values[-tail.numel():], tail)
