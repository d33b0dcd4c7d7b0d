"""The dense layer with bias, activation and residual (so3lr_b200.layers.linear) on the GPU,
against the plain formula in float64.

u is a type's unit roundoff (2^-8 bfloat16, 2^-11 float16, 2^-24 float32). A sum of k
products in float32 may be off by k ACC sum|x w| with ACC = 2^-22 (the tensor cores do not
promise round-to-nearest additions), at most; the 2-norm of what that and the roundings
make is held as well, where a bound over the whole sum would hide a lost term: two
independent roundings, 2 u relative. The activations' slopes are at most 1.13, their
arithmetic is off by 2^-20 (1 + |z|) at most (gelu: erff within 2 units of 1, times z; the
hardware's exponential and reciprocal in the others). z is kept for the gradient in the
element type: the slope is then off by u |z| times the second derivative, which times
|z| is below 0.6 for all of them but relu, whose slope a rounding does not change (a z
below the type's numbers aside).
"""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U32 = 2.0 ** -24
U = {torch.float32: U32, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
ACC, FUN = 2.0 ** -22, 2.0 ** -20
HALF = [torch.bfloat16, torch.float16]
ACTS = [None, "silu", "gelu", "gelu_tanh", "relu"]


@pytest.fixture(scope="module")
def layers():
    from so3lr_b200 import layers
    return layers


def _rand(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _act(z, act):
    """(value, slope) in float64"""
    if act is None:
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _within(got, want, bound, what):
    off = (got.double() - want).abs()
    over = (want.abs() + bound > torch.finfo(got.dtype).max) & torch.isinf(got) & (got.double().sign() == want.sign())
    bad = ~((off <= bound) | over)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, first at "
                                 f"{bad.nonzero()[0].tolist()}: {float(off[bad][0]):.3e} > {float(bound.expand_as(off)[bad][0]):.3e}")


def _norm_within(got, want, u, what):
    if want.numel() >= 64 and float(want.norm()) > 0 and bool(torch.isfinite(got).all()):
        rel = float((got.double() - want).norm() / want.norm())
        assert rel <= 2 * u, f"{what}: 2-norm off by {rel:.2e}"


def _make(rows, k, n, dtype, bias=None, residual=False, seed=0):
    return dict(x=_rand(seed + 1, rows, k, dtype=dtype), weight=_rand(seed + 2, n, k, dtype=dtype, scale=k ** -0.5),
                bias=None if bias is None else _rand(seed + 3, n, dtype=bias, scale=0.5),
                residual=_rand(seed + 4, rows, n, dtype=dtype) if residual else None)


def _sums(t):
    """z in float64 and the bound of its float32 error"""
    x, w = t["x"].double(), t["weight"].double()
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    if t["bias"] is not None:
        z, size = z + t["bias"].double(), size + t["bias"].double().abs()
    return z, (x.shape[1] + 1) * ACC * size


def _check(layers, t, act, what="", backward=True):
    dtype = t["x"].dtype
    u = U[dtype]
    z, err = _sums(t)
    value, slope = _act(z, act)
    r = t["residual"].double() if t["residual"] is not None else torch.zeros_like(z)
    want = value + r
    fun = 0.0 if act in (None, "relu") else FUN
    y = layers.linear(**t, activation=act)
    far = 1.2 * err + fun * (1 + z.abs()) + U32 * (value.abs() + r.abs())
    assert y.dtype == dtype and y.shape == want.shape
    _within(y, want, u * want.abs() + (1 + u) * far + TINY[dtype], what + " y")
    _norm_within(y, want, u, what + " y")
    if not backward:
        return y
    y2, saved = layers.linear_train(**t, activation=act)
    assert torch.equal(y, y2)
    dy = _rand(9, *want.shape, dtype=dtype)
    dx, dw, db = layers.linear_backward(dy, saved)
    d = dy.double()
    dz = d * slope
    # what the kept z's rounding, its float32 error and the slope's arithmetic make of dz, and dz's own rounding
    bend = 0.0 if act is None else 1.2
    loose = d.abs() * (bend * (u + err) + fun * (1 + z.abs())) if act != "relu" else \
        d.abs() * (z.abs() <= err + TINY[dtype]).double()
    rounded = loose + (u * (dz.abs() + loose) + TINY[dtype] if act is not None else 0.0)
    x, w = t["x"].double(), t["weight"].double()
    rows, n = dz.shape
    ref, size = dz @ w, (dz.abs() + rounded) @ w.abs()
    _within(dx, ref, u * ref.abs() + (1 + u) * (rounded @ w.abs() + n * ACC * size) + TINY[dtype], what + " dx")
    _norm_within(dx, ref, u, what + " dx")
    ref, size = dz.t() @ x, (dz.abs() + rounded).t() @ x.abs()
    _within(dw, ref, u * ref.abs() + (1 + u) * (rounded.t() @ x.abs() + rows * ACC * size) + TINY[dtype], what + " dw")
    _norm_within(dw, ref, u, what + " dw")
    if t["bias"] is None:
        assert db is None
    else:
        kind = t["bias"].dtype
        assert db.dtype == kind
        ref = dz.sum(0)
        _within(db, ref, U[kind] * ref.abs() + (1 + U[kind]) * (loose.sum(0) + (rows + 8) * U32 * (dz.abs() + loose).sum(0))
                + TINY[kind], what + " dbias")
    return y


SIZES = [(1, 1, 1), (1, 64, 8), (1, 2048, 512), (2, 7, 3), (16, 256, 256), (17, 100, 130), (5, 1003, 251), (33, 64, 72),
         (200, 256, 1024), (333, 1000, 1531), (257, 128, 8), (600, 8, 520), (1000, 251, 91), (300, 8192, 64), (129, 1, 129)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows, k, n", SIZES)
def test_forward_and_backward(layers, rows, k, n, dtype):
    for i, act in enumerate(ACTS):
        t = _make(rows, k, n, dtype, (None, dtype, torch.float32)[i % 3], residual=i % 2 == 0)
        _check(layers, t, act, f"{act}")


@pytest.mark.parametrize("act", ACTS)
def test_all_operands(layers, act):
    """Every activation with both types of bias, with and without a residual, in each kernel."""
    for rows in (3, 700):
        for bias in (None, torch.float32, torch.float16):
            for residual in (False, True):
                _check(layers, _make(rows, 192, 264, torch.float16, bias, residual), act, f"{rows} {bias} {residual}")


@pytest.mark.parametrize("rows, k, n", [(513, 4096, 300), (300, 20000, 256), (130, 70000, 40), (6000, 256, 320), (4000, 130, 2200)])
def test_split_contractions(layers, rows, k, n):
    """Tiles that are split along the contraction, forward and in either gradient."""
    for dtype, act in ((torch.bfloat16, "gelu_tanh"), (torch.float16, None)):
        _check(layers, _make(rows, k, n, dtype, torch.float32, True), act, f"{act}")


@pytest.mark.parametrize("shift", [0, 1, 3, 8])
def test_strides_and_alignments(layers, shift):
    """Operands inside wider rows and off the boundaries; a residual and an x of stride 0."""
    for rows, k, n in ((5, 96, 72), (300, 100, 130), (260, 256, 264)):
        def inside(v, i):
            wide = _rand(20 + i, v.shape[0], v.shape[1] + 40, dtype=v.dtype)
            return wide[:, shift:shift + v.shape[1]].copy_(v)
        t = _make(rows, k, n, torch.bfloat16, torch.bfloat16, True)
        for i, name in enumerate(("x", "weight", "residual")):
            t[name] = inside(t[name], i)
        bias = torch.zeros(n + 8, device="cuda", dtype=torch.bfloat16)
        t["bias"] = bias[shift % 8:shift % 8 + n].copy_(t["bias"])
        _check(layers, t, "silu", f"{rows}")
        dy = inside(_rand(9, rows, n, dtype=torch.bfloat16), 3)
        _, saved = layers.linear_train(**t, activation="silu")
        for a, b in zip(layers.linear_backward(dy, saved), layers.linear_backward(dy.contiguous(), saved)):
            assert torch.equal(a, b)
        t["residual"], t["x"] = t["residual"][:1].expand(rows, n), t["x"][:1].expand(rows, k)
        _check(layers, t, "gelu", f"{rows} broadcast", backward=False)


def test_leading_dimensions_and_no_rows(layers):
    t = _make(24, 96, 40, torch.bfloat16, torch.float32, True)
    y = layers.linear(**t, activation="relu")
    folded = dict(t, x=t["x"].view(2, 3, 4, 96), residual=t["residual"].view(2, 3, 4, 40))
    y4, saved = layers.linear_train(**folded, activation="relu")
    assert y4.shape == (2, 3, 4, 40) and torch.equal(y4.view(24, 40), y)
    dx, _, _ = layers.linear_backward(y4, saved)
    assert dx.shape == (2, 3, 4, 96)
    t = _make(0, 96, 40, torch.bfloat16, torch.float32, True)
    y, saved = layers.linear_train(**t, activation="relu")
    dx, dw, db = layers.linear_backward(y, saved)
    assert y.shape == (0, 40) and dx.shape == (0, 96) and bool((dw == 0).all()) and bool((db == 0).all())


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("act", ACTS[1:])
def test_activations_over_their_range(layers, act, dtype):
    """x = z through a weight of 1: values and gradients from the smallest to the largest of the type,
    a float16 sum beyond it, infinities and NaN."""
    finfo = torch.finfo(dtype)
    grid = torch.logspace(-6, math.log10(min(finfo.max, 1e30)) - 0.01, 4000, dtype=torch.float64, device="cuda")
    near = torch.linspace(-12, 12, 4001, dtype=torch.float64, device="cuda")
    x = torch.cat([grid, -grid, near, torch.zeros(1, device="cuda")]).to(dtype)[:, None]
    for rows in (x, x[:13]):
        w = torch.ones(1, 1, device="cuda", dtype=dtype)
        y, saved = layers.linear_train(rows, w, activation=act)
        z = rows.double()
        want, slope = _act(z, act)
        if act == "gelu_tanh":  # the powers of a far z are beyond float64's too
            slope = torch.where(z.abs() > 1e3, (z > 0).double(), slope)
        _within(y, want, U[dtype] * want.abs() + FUN * z.abs().clamp(max=16) + TINY[dtype], "y")
        dx, _, _ = layers.linear_backward(torch.ones_like(y), saved)
        _within(dx, slope, 2 * U[dtype] * slope.abs() + FUN * (1 + z.abs().clamp(max=16)) + TINY[dtype], "slope")
    if dtype == torch.float16:  # a sum beyond it: y is infinite or 0, the slope its limit. (Twice bfloat16's
        # largest is beyond float32 too, and z sigmoid(z) of minus infinity -inf * 0.)
        big = torch.tensor([[finfo.max], [-finfo.max]], device="cuda", dtype=dtype)
        w = torch.full((1, 1), 2.0, device="cuda", dtype=dtype)
        y, saved = layers.linear_train(big, w, activation=act)
        dx, _, _ = layers.linear_backward(torch.ones_like(y), saved)
        assert float(y[0]) == math.inf and float(y[1]) == 0.0
        assert float(dx[0]) == 2.0 and float(dx[1]) == 0.0
    nan = torch.full((20, 8), float("nan"), device="cuda", dtype=dtype)
    for rows in (nan[:3], nan):
        y, saved = layers.linear_train(rows, torch.ones(9, 8, device="cuda", dtype=dtype), activation=act)
        assert bool(torch.isnan(y).all())
        assert bool(torch.isnan(layers.linear_backward(torch.ones_like(y), saved)[0]).all())


def test_rows_do_not_mix(layers):
    """An infinity or a NaN in one row, channel or residual stays in it."""
    for rows in (9, 300):
        t = _make(rows, 128, 96, torch.bfloat16, torch.float32, True)
        clean = layers.linear(**t, activation="silu")
        t["x"][2, 5], t["weight"][7, 3], t["residual"][4, 6] = float("inf"), float("nan"), float("-inf")
        y = layers.linear(**t, activation="silu")
        same = torch.ones(rows, 96, dtype=torch.bool, device="cuda")
        same[2], same[:, 7], same[4, 6] = False, False, False
        assert torch.equal(y[same], clean[same])
        assert bool(torch.isnan(y[:, 7]).all()) and float(y[4, 6]) == -math.inf


def test_gradient_against_differences(layers):
    """Directional differences of the formula in float64, central, step 1e-6 of values near 1: off by
    about 1e-9 relative. Compared with the gradients in float16 within the bounds that _check holds,
    taken along the direction; here their sum over all elements is taken as independent, 8 times the
    2-norm."""
    t = _make(40, 48, 56, torch.float16, torch.float32, True)
    dy = _rand(9, 40, 56, dtype=torch.float16)
    for act in ACTS:
        if act == "relu":
            continue  # not differentiable where differences would step over 0
        _, saved = layers.linear_train(**t, activation=act)
        got = dict(zip(("x", "weight", "bias"), layers.linear_backward(dy, saved)))
        d = {k: v.double() for k, v in t.items()}
        loss = lambda v: float((_act(v["x"] @ v["weight"].t() + v["bias"], act)[0] * dy.double()).sum())  # noqa: E731
        for i, (k, g) in enumerate(got.items()):
            way = _rand(30 + i, *g.shape).double()
            slope = (loss({**d, k: d[k] + 1e-6 * way}) - loss({**d, k: d[k] - 1e-6 * way})) / 2e-6
            value = float((g.double() * way).sum())
            bound = 8 * 3 * U[torch.float16] * float((g.double() * way).norm()) + 1e-6 * abs(slope) + 1e-6
            assert abs(value - slope) <= bound, (act, k, value, slope, bound)


def test_autograd(layers):
    for act in ACTS:
        t = {k: v.requires_grad_() for k, v in _make(50, 64, 96, torch.bfloat16, torch.float32, True).items()}
        y = layers.linear(**t, activation=act)
        dy = _rand(9, 50, 96, dtype=torch.bfloat16)
        got = torch.autograd.grad(y, list(t.values()), dy, retain_graph=True)
        plain = {k: v.detach() for k, v in t.items()}
        y2, saved = layers.linear_train(**plain, activation=act)
        assert torch.equal(y, y2)
        for a, b in zip(got, layers.linear_backward(dy, saved) + (dy,)):
            assert torch.equal(a, b)
        for k in t:  # each by itself
            only = dict(plain, **{k: t[k]})
            g, = torch.autograd.grad(layers.linear(**only, activation=act), t[k], dy)
            assert torch.equal(g, got[list(t).index(k)])
        # a gradient as autograd makes it: expanded, transposed
        g, = torch.autograd.grad(layers.linear(**t, activation=act).sum(), t["x"])
        want = layers.linear_backward(torch.ones_like(dy), saved)[0]
        assert torch.equal(g, want)
    with torch.no_grad():
        assert not layers.linear(**t).requires_grad


def test_in_place_and_captured(layers):
    """A captured training step, replayed on other data, on another stream."""
    t = _make(300, 128, 256, torch.bfloat16, torch.float32, True)
    dy = _rand(9, 300, 256, dtype=torch.bfloat16)

    def both():
        y, saved = layers.linear_train(**t, activation="gelu")
        return (y,) + layers.linear_backward(dy, saved)

    both()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both()
    for _ in range(3):
        t["x"].mul_(-0.5)
        torch.cuda.synchronize()
        want = both()
        with torch.cuda.stream(torch.cuda.Stream()):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, captured))


def test_calls_back_to_back(layers):
    """What a call reads, the call just before it may still be writing."""
    for rows, width in ((4, 256), (300, 200), (700, 256)):
        w = [_rand(40 + i, width, width, dtype=torch.bfloat16, scale=width ** -0.5) for i in range(6)]
        x = _rand(1, rows, width, dtype=torch.bfloat16)

        def chain(sync):
            h, kept = x, []
            for i in range(6):
                h, saved = layers.linear_train(h, w[i], None, h, activation="silu")
                kept.append(saved)
                if sync:
                    torch.cuda.synchronize()
            g, out = h, []
            for saved in reversed(kept):
                g, dw, _ = layers.linear_backward(g, saved)
                out.append(dw)
                if sync:
                    torch.cuda.synchronize()
            return [h, g] + out

        apart = chain(True)
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(apart, chain(False)))


def test_refusals(layers):
    from so3lr_b200 import So3lrError

    def refused(match, kind=ValueError, act=None, **change):
        with pytest.raises(kind, match=match):
            layers.linear(**{**_make(4, 32, 24, torch.bfloat16, torch.float32, True), **change}, activation=act)

    zeros = lambda *s, t=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=t)  # noqa: E731
    refused("no CPU path", x=torch.zeros(4, 32))
    refused("x must be one of", x=zeros(4, 32, t=torch.float32))
    refused("weight must be torch.bfloat16", weight=zeros(24, 32, t=torch.float16))
    refused("weight must have rows of 32", weight=zeros(24, 31))
    refused("weight must have at least one row", weight=zeros(0, 32))
    refused("bias must be a 1-D", bias=zeros(23))
    refused("bias must be torch.bfloat16 or torch.float32", bias=zeros(24, t=torch.float16))
    refused("residual must have the shape", residual=zeros(4, 23))
    refused("residual must be torch.bfloat16", residual=zeros(4, 24, t=torch.float16))
    refused("activation must be one of", act="tanh")
    refused("activation must be one of", act=3)
    refused("contiguous last dimension", x=zeros(32, 4).t())
    y, saved = layers.linear_train(**_make(4, 32, 24, torch.bfloat16), activation="silu")
    with pytest.raises(ValueError, match="dy must have rows of 24"):
        layers.linear_backward(y[:, :23].contiguous(), saved)
    with pytest.raises(ValueError, match="saved"):
        layers.linear_backward(y, saved[:2] + (None,) + saved[3:])
    with pytest.raises(So3lrError, match="k must be in"):
        wide = zeros(1, 1 << 20 | 1)
        layers.linear(wide, wide)
    with torch.autograd.forward_ad.dual_level():
        x = zeros(4, 32)
        refused("forward-mode tangent", x=torch.autograd.forward_ad.make_dual(x, x))
