"""The norms on both sides of a block (so3lr_b200.layers.sandwich_norm) on the GPU, against
the plain formula in float64.

u is a type's unit roundoff (2^-8 bfloat16, 2^-11 float16, 2^-24 float32). Everything
between the inputs and a result is float32: F32 = 64 u of float32 covers a chain of
statistics (16 + 5 + 32 additions, a few products) relative to the sum of the magnitudes
that meet in it; a result is rounded to its type once. The second norm and the gradients
are those of the s that was stored, so its rounding does not count in them. Sums over
rows: one float32 rounding for each row besides.
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U32 = 2.0 ** -24
U = {torch.float32: U32, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
F32 = 64 * U32
EPS = 1e-6


@pytest.fixture(scope="module")
def layers():
    from so3lr_b200 import layers
    return layers


def _rand(seed, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def _within(got, want, bound, what):
    off = (got.double() - want).abs()
    # beyond the type's largest number the rounding is the infinity of that sign (rows of zeros have
    # gradients of 1e6, float16 ends at 65504)
    over = (want.abs() + bound > torch.finfo(got.dtype).max) & torch.isinf(got) & (got.double().sign() == want.sign())
    bad = ~((off <= bound) | over)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, first at "
                                 f"{bad.nonzero()[0].tolist()}: {float(off[bad][0]):.3e}")


def _inputs(rows, width, dtype, wdtype=None, gate=True, scale=True, seed=0):
    wdtype = wdtype or dtype
    return dict(x=_rand(seed + 1, rows, width, dtype=dtype, scale=0.7),
                residual=_rand(seed + 2, rows, width, dtype=dtype, scale=2.0),
                weight=_rand(seed + 3, width, dtype=wdtype, scale=0.2, shift=0.5),
                next_weight=_rand(seed + 4, width, dtype=wdtype, scale=0.2, shift=1.0),
                gate=_rand(seed + 5, rows, width, dtype=dtype, shift=0.5) if gate else None,
                residual_scale=_rand(seed + 6, width, dtype=wdtype, scale=0.1, shift=1.0) if scale else None)


def _double(t):
    return {k: None if v is None else v.double() for k, v in t.items()}


def _check_forward(y, s, t, eps=EPS):
    d, dtype = _double(t), t["x"].dtype
    gate = 1.0 if d["gate"] is None else d["gate"]
    scale = 1.0 if d["residual_scale"] is None else d["residual_scale"]
    rx = 1.0 / ((d["x"] ** 2).mean(1, keepdim=True) + eps).sqrt()
    added, kept = gate * d["x"] * rx * d["weight"], d["residual"] * scale
    _within(s, added + kept, U[dtype] * (added + kept).abs() + F32 * (added.abs() + kept.abs()) + TINY[dtype], "s")
    f = s.double()
    ref = f / ((f ** 2).mean(1, keepdim=True) + eps).sqrt() * d["next_weight"]
    _within(y, ref, (U[dtype] + F32) * ref.abs() + TINY[dtype], "y")


def _gradients(t, s, dy, ds, eps=EPS):
    """{name: (gradient, what its float32 error is relative to)}"""
    d, s, dy = _double(t), s.double(), dy.double()
    ds = torch.zeros_like(s) if ds is None else ds.double()
    gate = torch.ones_like(s) if d["gate"] is None else d["gate"]
    scale = torch.ones_like(s[0]) if d["residual_scale"] is None else d["residual_scale"]
    mean = lambda v: v.mean(1, keepdim=True)  # noqa: E731
    rx, rs = 1.0 / (mean(d["x"] ** 2) + eps).sqrt(), 1.0 / (mean(s ** 2) + eps).sqrt()
    xh, sh, a2 = d["x"] * rx, s * rs, dy * d["next_weight"]
    g = rs * (a2 - sh * mean(a2 * sh)) + ds
    big = rs * (a2.abs() + sh.abs() * mean((a2 * sh).abs())) + ds.abs()
    q, w = g * gate, d["weight"]
    a1, big1 = q * w, big * (gate * w).abs()
    out = dict(dx=(rx * (a1 - xh * mean(a1 * xh)), rx * (big1 + xh.abs() * mean(big1 * xh.abs()))),
               dresidual=(g * scale, big * scale.abs()), dweight=((q * xh).sum(0), (big * (gate * xh).abs()).sum(0)),
               dnext_weight=((dy * sh).sum(0), (dy * sh).abs().sum(0)))
    if d["gate"] is not None:
        out["dgate"] = g * xh * w, big * (xh * w).abs()
    if d["residual_scale"] is not None:
        out["dresidual_scale"] = (g * d["residual"]).sum(0), (big * d["residual"].abs()).sum(0)
    return out


def _check_backward(got, t, s, dy, ds, eps=EPS):
    names = ("dx", "dresidual", "dweight", "dnext_weight", "dgate", "dresidual_scale")
    want = _gradients(t, s, dy, ds, eps)
    rows, dtype = s.shape[0], t["x"].dtype
    for name, value in zip(names, got):
        if name not in want:
            assert value is None, name
            continue
        ref, size = want[name]
        over_rows = ref.dim() == 1
        kind = t["weight"].dtype if over_rows else dtype
        assert value.dtype == kind and value.shape == ref.shape, name
        rel = (rows * U32 + 2 * F32) if over_rows else 2 * F32
        _within(value, ref, U[kind] * ref.abs() + rel * size + TINY[kind], name)


SIZES = [(1, 1), (1, 2048), (3, 7), (5, 64), (40, 65), (5, 128), (2, 511), (9, 512), (4, 513), (7, 1003), (700, 256),
         (3, 4096), (2, 4097), (600, 1003), (2, 8192), (2, 8200), (2, 16384), (3, 16383)]


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("rows, width", SIZES)
def test_forward_and_backward(layers, rows, width, dtype):
    for wdtype, gate, scale in ((dtype, True, True), (torch.float32, False, True), (dtype, True, False),
                                (torch.float32, False, False)):
        t = _inputs(rows, width, dtype, wdtype, gate, scale)
        y, s = layers.sandwich_norm(**t, eps=EPS)
        _check_forward(y, s, t)
        dy, ds = _rand(7, rows, width, dtype=dtype), _rand(8, rows, width, dtype=dtype) if gate else None
        _check_backward(layers.sandwich_norm_backward(dy, ds, s, **t, eps=EPS), t, s, dy, ds)


@pytest.mark.parametrize("dtype", list(U))
def test_many_rows(layers, dtype):
    """Blocks that walk over many rows, the last of them fewer."""
    for rows, width in ((5003, 64), (5003, 72), (4001, 128), (3001, 250), (3001, 256), (2003, 512), (1501, 768),
                        (1203, 1024), (1201, 1003), (700, 4096), (401, 8192)):
        t = _inputs(rows, width, dtype)
        y, s = layers.sandwich_norm(**t, eps=EPS)
        _check_forward(y, s, t)
        dy, ds = _rand(7, rows, width, dtype=dtype), _rand(8, rows, width, dtype=dtype)
        _check_backward(layers.sandwich_norm_backward(dy, ds, s, **t, eps=EPS), t, s, dy, ds)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignments(layers, dtype):
    """Rows inside wider ones, off the boundaries, tensors that lie differently, gates of a stride of 0."""
    for rows, width, shifts in ((33, 256, (0,) * 8), (33, 256, (1,) * 8), (33, 256, (3, 0, 1, 2, 5, 0, 0, 0)),
                                (9, 1000, (8,) * 8), (9, 1003, (1, 2, 3, 4, 5, 6, 7, 8)), (5, 5000, (1,) * 8)):
        def inside(k, i, row):
            wide = _rand(20 + i, rows, width + 40, dtype=dtype)
            return wide[:, shifts[i]:shifts[i] + width].copy_(row)
        t = _inputs(rows, width, dtype)
        for i, k in enumerate(("x", "residual", "gate")):
            t[k] = inside(k, i, t[k])
        y, s = layers.sandwich_norm(**t, eps=EPS)
        _check_forward(y, s, t)
        dy, ds = inside("dy", 3, _rand(7, rows, width, dtype=dtype)), inside("ds", 4, _rand(8, rows, width, dtype=dtype))
        s = inside("s", 5, s)
        _check_backward(layers.sandwich_norm_backward(dy, ds, s, **t, eps=EPS), t, s, dy, ds)
        t["gate"] = t["gate"][:1].expand(rows, width)
        y, s = layers.sandwich_norm(**t, eps=EPS)
        _check_forward(y, s, t)


def test_leading_dimensions_and_no_rows(layers):
    t = _inputs(24, 96, torch.bfloat16)
    y, s = layers.sandwich_norm(**t)
    folded = {k: v.view(2, 3, 4, 96) if v.dim() == 2 else v for k, v in t.items()}
    y4, s4 = layers.sandwich_norm(**folded)
    assert y4.shape == (2, 3, 4, 96) and torch.equal(y4.view(24, 96), y) and torch.equal(s4.view(24, 96), s)
    t = _inputs(0, 96, torch.bfloat16)
    y, s = layers.sandwich_norm(**t)
    assert y.shape == s.shape == (0, 96)
    out = layers.sandwich_norm_backward(y, s, s, **t)
    assert out[0].shape == out[1].shape == out[4].shape == (0, 96)
    assert all(bool((out[i] == 0).all()) for i in (2, 3, 5))


def test_special_rows(layers):
    """Zeros, infinities and NaN stay in their rows; eps = 0 and a row of zeros is 0 / 0."""
    for dtype in U:
        for width in (100, 256, 1003, 4096):
            t = _inputs(8, width, dtype)
            t["x"][1] = 0
            t["x"][2, 5] = float("inf")
            t["residual"][3, 7] = float("nan")
            t["gate"][4, 3] = float("-inf")
            t["x"][5], t["residual"][5] = 0, 0
            good = torch.tensor([0, 1, 5, 6, 7], device="cuda")
            y, s = layers.sandwich_norm(**t, eps=EPS)
            part = {k: v[good] if v.dim() == 2 else v for k, v in t.items()}
            _check_forward(y[good], s[good], part)
            assert bool((y[5] == 0).all())
            for r in (2, 3, 4):
                assert bool(torch.isnan(y[r]).any())
            dy, ds = _rand(7, 8, width, dtype=dtype), _rand(8, 8, width, dtype=dtype)
            out = layers.sandwich_norm_backward(dy, ds, s, **t, eps=EPS)
            want = _gradients(part, s[good], dy[good], ds[good])
            for i, name in ((0, "dx"), (1, "dresidual"), (4, "dgate")):
                ref, size = want[name]
                _within(out[i][good], ref, U[dtype] * ref.abs() + 2 * F32 * size + TINY[dtype], name)
            y, _ = layers.sandwich_norm(**t, eps=0.0)
            assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[5]).all())


def test_gradient_against_differences(layers):
    """Directional differences of the formula in float64, central, step 1e-5: off by about 1e-10 of
    what they are taken of, which the float32 bounds cover many times."""
    rows, width = 4, 37
    t = _inputs(rows, width, torch.float32)
    dy, ds = _rand(7, rows, width), _rand(8, rows, width)
    _, s = layers.sandwich_norm(**t, eps=EPS)
    got = layers.sandwich_norm_backward(dy, ds, s, **t, eps=EPS)
    want = _gradients(t, s, dy, ds)

    def loss(d):
        norm = lambda v, w: v / ((v * v).mean(1, keepdim=True) + EPS).sqrt() * w  # noqa: E731
        s = d["residual"] * d["residual_scale"] + d["gate"] * norm(d["x"], d["weight"])
        return float((norm(s, d["next_weight"]) * dy.double()).sum() + (s * ds.double()).sum())

    names = dict(x="dx", residual="dresidual", weight="dweight", next_weight="dnext_weight", gate="dgate",
                 residual_scale="dresidual_scale")
    order = ("dx", "dresidual", "dweight", "dnext_weight", "dgate", "dresidual_scale")
    for i, (k, name) in enumerate(names.items()):
        way, d = _rand(30 + i, *t[k].shape).double(), _double(t)
        moved = [loss({**d, k: d[k] + h * way}) for h in (1e-5, -1e-5)]
        slope = (moved[0] - moved[1]) / 2e-5
        value = float((got[order.index(name)].double() * way).sum())
        ref, size = want[name]
        # s as stored is a rounding (u of float32) away from the formula's: as much as the statistics are off
        bound = float(((U32 * ref.abs() + 4 * F32 * size) * way.abs()).sum()) + 1e-7 * abs(slope)
        assert abs(value - slope) <= bound, (name, value, slope, bound)


def test_autograd(layers):
    """Gradients through the recorded call, outputs that nothing reads, a broadcast gate, and a second use."""
    rows, width = 50, 96
    for wdtype in (torch.float32, torch.bfloat16):
        t = {k: v.requires_grad_() for k, v in _inputs(rows, width, torch.bfloat16, wdtype).items()}
        y, s = layers.sandwich_norm(**t)
        dy, ds = _rand(7, rows, width, dtype=torch.bfloat16), _rand(8, rows, width, dtype=torch.bfloat16)
        zeros = torch.zeros_like(dy)
        plain = {k: v.detach() for k, v in t.items()}
        for outs, grads, used in (((y, s), (dy, ds), (dy, ds)), ((y,), (dy,), (dy, None)), ((s,), (ds,), (zeros, ds))):
            got = torch.autograd.grad(outs, list(t.values()), grads, retain_graph=True)
            want = layers.sandwich_norm_backward(used[0], used[1], s.detach(), **plain)
            order = (0, 1, 2, 3, 4, 5)
            for g, i in zip(got, order):
                assert torch.equal(g, want[i])
    gate = torch.randn(1, width, device="cuda").bfloat16().requires_grad_()
    t = _inputs(rows, width, torch.bfloat16)
    plain = dict(t, gate=gate.detach().expand(rows, width))
    y, s = layers.sandwich_norm(**dict(t, gate=gate.expand(rows, width)))
    dgate, = torch.autograd.grad(y, gate, dy)
    want = layers.sandwich_norm_backward(dy, None, s.detach(), **plain)[4]
    assert torch.equal(dgate, want.sum(0, keepdim=True))
    with torch.no_grad():
        assert not layers.sandwich_norm(**dict(t, gate=gate.expand(rows, width)))[0].requires_grad


def test_captured_and_on_another_stream(layers):
    rows, width = 300, 1024
    t = _inputs(rows, width, torch.bfloat16)
    dy, ds = _rand(7, rows, width, dtype=torch.bfloat16), _rand(8, rows, width, dtype=torch.bfloat16)

    def both():
        y, s = layers.sandwich_norm(**t)
        return (y, s) + layers.sandwich_norm_backward(dy, ds, s, **t)

    both()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both()
    for k in range(3):
        t["x"].mul_(-0.5)
        torch.cuda.synchronize()
        want = both()
        with torch.cuda.stream(torch.cuda.Stream()):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, captured))


def test_calls_back_to_back(layers):
    """A call reads what the one just before it wrote; the column sums what their rows' kernel did."""
    for rows, width in ((700, 96), (600, 1003), (900, 2048), (100, 6000)):
        t = _inputs(rows, width, torch.float32)
        dy = _rand(7, rows, width)
        apart, together = [], []
        for k in range(6):
            y, s = layers.sandwich_norm(**t)
            torch.cuda.synchronize()
            apart.append(layers.sandwich_norm_backward(dy * 2.0 ** k, None, s, **t)[2:])
            torch.cuda.synchronize()
        scaled = [dy * 2.0 ** k for k in range(6)]
        for k in range(6):
            y, s = layers.sandwich_norm(**t)
            together.append(layers.sandwich_norm_backward(scaled[k], None, s, **t)[2:])
        for a, b in zip(apart, together):
            assert all(torch.equal(x, z) for x, z in zip(a, b))


def test_refusals(layers):
    from so3lr_b200 import So3lrError

    def refused(match, kind=ValueError, **change):
        with pytest.raises(kind, match=match):
            layers.sandwich_norm(**{**_inputs(4, 32, torch.bfloat16), **change})

    half, ones = torch.zeros(4, 32, device="cuda", dtype=torch.float16), torch.ones(32, device="cuda")
    refused("no CPU path", x=torch.zeros(4, 32))
    refused("x must be one of", x=torch.zeros(4, 32, device="cuda", dtype=torch.int32))
    refused("residual must have the shape", residual=torch.zeros(3, 32, device="cuda", dtype=torch.bfloat16))
    refused("residual must be torch.bfloat16", residual=half)
    refused("gate must have the shape", gate=torch.zeros(4, 1, device="cuda", dtype=torch.bfloat16))
    refused("gate must be torch.bfloat16", gate=half)
    refused("gate must have a contiguous last", gate=torch.zeros(4, 1, device="cuda", dtype=torch.bfloat16).expand(4, 32))
    refused("weight must be a 1-D", weight=ones[:31])
    refused("next_weight must be torch.bfloat16", next_weight=ones)
    refused("residual_scale must be torch.bfloat16", residual_scale=ones)
    refused("residual must be a tensor", residual=None)
    refused("eps", kind=So3lrError, eps=-1.0)
    wide = _inputs(1, 16385, torch.bfloat16)
    with pytest.raises(So3lrError, match="width must be in"):
        layers.sandwich_norm(**wide)
    with torch.autograd.forward_ad.dual_level():
        x = torch.zeros(4, 32, device="cuda", dtype=torch.bfloat16)
        refused("forward-mode tangent", x=torch.autograd.forward_ad.make_dual(x, x))
