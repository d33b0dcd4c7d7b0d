"""Row-wise feed-forward layers (so3lr_b200.layers) on the GPU, against plain
float64 formulas written here.

Tolerances are bounds, not fits. u is the unit roundoff of a type (2^-8 bfloat16,
2^-11 float16, 2^-24 float32). A result that the kernel computes in float32 and
rounds once may be off by u |result| plus the float32 error of what it was
computed from; sums of n products in float32 may be off by n ACC sum|a b| with
ACC = 2^-22 (the tensor cores do not promise round-to-nearest additions, so four
times the unit roundoff is allowed for each). Where a bound over the whole sum
would hide a lost term, the 2-norm of the error is held as well: two independent
roundings to the type, 2 u relative.
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}  # half a subnormal step
F32 = 64 * 2.0 ** -24  # float32 statistics: at most 16 + 5 + 32 additions in a chain, and a few products
ACC = 2.0 ** -22
EPS = 1e-6
HALF = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def layers():
    from so3lr_b200 import layers
    return layers


def _rand(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _within(got, want, bound, what):
    bad = (got.double() - want).abs() > bound
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, first at {bad.nonzero()[0].tolist()}"


def _norm_ref(s, w, eps=EPS):
    rstd = 1.0 / torch.sqrt((s * s).mean(1, keepdim=True) + eps)
    return s * rstd * w, rstd


# ------------------------------------------------------------------------ norm
NORM_SIZES = [(1, 1), (1, 2048), (3, 7), (5, 128), (2, 511), (9, 512), (4, 513), (7, 1003), (300, 256), (2, 8192),
              (2, 16384), (3, 16383)]


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("rows, width", NORM_SIZES)
def test_rms_norm_forward_and_backward(layers, rows, width, dtype):
    for wdtype, with_residual in ((dtype, True), (torch.float32, False)):
        x, r = _rand(1, rows, width, dtype=dtype), _rand(2, rows, width, dtype=dtype, scale=2.0)
        w = (1 + 0.1 * _rand(3, width)).to(wdtype)
        y, s = layers.rms_norm(x, w, r if with_residual else None, eps=EPS)
        want_s = (x.float() + r.float()).to(dtype) if with_residual else x
        assert torch.equal(s, want_s)
        ref, rstd = _norm_ref(s.double(), w.double())
        _within(y, ref, (U[dtype] + F32) * ref.abs() + TINY[dtype], "y")

        dy, ds = _rand(4, rows, width, dtype=dtype), _rand(5, rows, width, dtype=dtype)
        dx, dw = layers.rms_norm_backward(dy, s, w, ds if with_residual else None, eps=EPS)
        xh, a = s.double() * rstd, dy.double() * w.double()
        rest = ds.double() if with_residual else torch.zeros_like(a)
        ref = rstd * (a - xh * (a * xh).mean(1, keepdim=True)) + rest
        size = rstd * (a.abs() + xh.abs() * (a * xh).abs().mean(1, keepdim=True)) + rest.abs()
        _within(dx, ref, U[dtype] * ref.abs() + F32 * size + TINY[dtype], "dx")
        ref, size = (dy.double() * xh).sum(0), (dy.double() * xh).abs().sum(0)
        _within(dw, ref, U[wdtype] * ref.abs() + (rows * 2.0 ** -24 + F32) * size + TINY[wdtype], "dweight")


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("rows, width", NORM_SIZES)
def test_rms_norm_int8(layers, rows, width, dtype):
    x, r, w = _rand(1, rows, width, dtype=dtype), _rand(2, rows, width, dtype=dtype), 1 + 0.1 * _rand(3, width)
    codes, scales, s = layers.rms_norm_int8(x, w, r, eps=EPS)
    assert codes.shape == (rows, width) and codes.dtype == torch.int8 and codes.stride(0) % 16 == 0
    ref, _ = _norm_ref(s.double(), w.double())
    _check_codes(codes, scales, ref)
    y = layers.dequantize_int8(codes, scales, dtype)
    want = codes.float() * scales[:, None]
    assert torch.equal(y, want.to(dtype))


def _check_codes(codes, scales, ref):
    want = ref.abs().amax(1) / 127
    _within(scales, want, F32 * want + 2.0 ** -126, "scales")
    # half a step, and what the float32 value may be off by
    step = scales.double()[:, None]
    _within(codes.double() * step, ref, step * (0.5 + 127 * 2 * F32) + 2.0 ** -120, "values")
    live = want > 2.0 ** -120
    assert bool((codes.abs().amax(1)[live] == 127).all())


def test_rms_norm_special_rows(layers):
    for dtype in U:
        for width in (100, 256, 1003, 4096):
            x = _rand(1, 6, width, dtype=dtype)
            x[1] = 0
            x[2, 5] = float("inf")
            x[3, 7] = float("nan")
            x[4, 3] = -float("inf")
            w = torch.ones(width, device="cuda")
            y, s = layers.rms_norm(x, w, eps=EPS)
            assert s is x
            ref, _ = _norm_ref(x.double(), w.double())
            assert torch.equal(torch.isnan(y), torch.isnan(ref))
            assert bool((y[1] == 0).all())
            codes, scales, _ = layers.rms_norm_int8(x, w, eps=EPS)
            assert float(scales[1]) == 0 and bool((codes[1] == 0).all())
            assert bool(torch.isnan(scales[2:5]).all()) and bool((codes[2:5] == 0).all())
            good = torch.tensor([0, 5], device="cuda")
            _check_codes(codes[good], scales[good], ref[good])
            assert bool(torch.isnan(layers.dequantize_int8(codes, scales)[2:5]).all())
            # eps = 0 and a row of zeros: 0 / 0, as the formula has it
            y0, _ = layers.rms_norm(x[:2], w, eps=0.0)
            assert bool(torch.isnan(y0[1]).all()) and bool(torch.isfinite(y0[0]).all())


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("rows, width, with_residual", [(2501, 904, False), (3001, 520, True), (2600, 4096, True),
                                                        (2400, 8192, False), (5003, 1536, False)])
def test_rms_norm_int8_of_many_rows(layers, rows, width, with_residual, dtype):
    """Blocks that walk over rows, with rows of zeros, infinities and NaN, large and small ones among them."""
    x, w = _rand(1, rows, width, dtype=dtype), 1 + 0.1 * _rand(3, width)
    r = _rand(2, rows, width, dtype=dtype) if with_residual else None
    kinds = torch.arange(rows, device="cuda") % 11
    for t in (x,) if r is None else (x, r):
        t[kinds == 3] = 0
        t[kinds == 7] *= 2.0 ** 12 if dtype is torch.float16 else 2.0 ** 50
        t[kinds == 8] *= 2.0 ** -9
    x[kinds == 4, width - 1] = float("inf")
    x[kinds == 5, 0] = float("nan")
    codes, scales, s = layers.rms_norm_int8(x, w, r, eps=EPS)
    want_s = x if r is None else (x.float() + r.float()).to(dtype)
    assert torch.equal(s.nan_to_num(nan=1.0), want_s.nan_to_num(nan=1.0))
    lost = (kinds == 4) | (kinds == 5)
    assert bool(torch.isnan(scales[lost]).all()) and bool((codes[lost] == 0).all())
    assert bool((scales[kinds == 3] == 0).all()) and bool((codes[kinds == 3] == 0).all())
    ref, _ = _norm_ref(s[~lost].double(), w.double())
    _check_codes(codes[~lost], scales[~lost], ref)


def test_rms_norm_layouts(layers):
    """Views: odd offsets, row strides, broadcast rows, leading dimensions, no rows."""
    big = _rand(1, 20, 300, dtype=torch.bfloat16)
    w = 1 + 0.1 * _rand(2, 264)
    for x in (big[:, 3:267], big[::3, :264], big[:1, :264].expand(9, 264), big[:, 8:272]):
        r = _rand(3, *x.shape, dtype=torch.bfloat16)
        y, s = layers.rms_norm(x, w, r)
        y2, s2 = layers.rms_norm(x.contiguous(), w, r)
        assert torch.equal(s, s2)
        ref, _ = _norm_ref(s.double(), w.double())
        _within(y, ref, (U[torch.bfloat16] + F32) * ref.abs(), "y")
        dx, dw = layers.rms_norm_backward(y, x, w)
        dx2, dw2 = layers.rms_norm_backward(y, x.contiguous(), w)
        _within(dx, dx2.double(), 2 * U[torch.bfloat16] * (dx2.double().abs() + 1e-3), "dx of a view")
        _within(dw, dw2.double(), 1e-4 * dw2.double().abs().max(), "dweight of a view")
    x3 = _rand(4, 2, 5, 264)
    y3, s3 = layers.rms_norm(x3, w, x3)
    assert y3.shape == x3.shape and s3.shape == x3.shape
    assert torch.equal(y3.view(10, 264), layers.rms_norm(x3.view(10, 264), w, x3.view(10, 264))[0])
    none = big[:0, :264]
    y0, s0 = layers.rms_norm(none, w, none)
    assert y0.shape == (0, 264) and s0.shape == (0, 264)
    dx, dw = layers.rms_norm_backward(none, none, w)
    assert dx.shape == (0, 264) and bool((dw == 0).all())


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("rows, width, offset", [(40, 63, 0), (19, 130, 1), (33, 257, 0), (50, 515, 3), (600, 1027, 2),
                                                 (5, 4099, 5), (3, 8187, 1), (2, 16383, 1)])
def test_rms_norm_rows_off_the_boundaries(layers, rows, width, offset, dtype):
    """Rows that all start equally far past a boundary, and tensors that differ in it."""
    def view(seed, apart=0):
        return _rand(seed, rows * width + offset + apart, dtype=dtype)[offset + apart:].view(rows, width)

    for apart in (0, 1):
        x, r, dy, ds = view(1), view(2, apart), view(3), view(4, apart)
        w = (1 + 0.1 * _rand(5, width + 1)[1:]).contiguous()
        y, s = layers.rms_norm(x, w, r)
        assert torch.equal(s, (x.float() + r.float()).to(dtype))
        ref, rstd = _norm_ref(s.double(), w.double())
        _within(y, ref, (U[dtype] + F32) * ref.abs() + TINY[dtype], "y")
        codes, scales, s8 = layers.rms_norm_int8(x, w, r)
        assert torch.equal(s8, s)
        _check_codes(codes, scales, ref)
        assert torch.equal(layers.dequantize_int8(codes, scales, dtype), (codes.float() * scales[:, None]).to(dtype))
        sv = view(6)
        dx, dw = layers.rms_norm_backward(dy, sv, w, ds)
        _, rstd = _norm_ref(sv.double(), w.double())
        xh, a = sv.double() * rstd, dy.double() * w.double()
        want = rstd * (a - xh * (a * xh).mean(1, keepdim=True)) + ds.double()
        size = rstd * (a.abs() + xh.abs() * (a * xh).abs().mean(1, keepdim=True)) + ds.double().abs()
        _within(dx, want, U[dtype] * want.abs() + F32 * size + TINY[dtype], "dx")
        want, size = (dy.double() * xh).sum(0), (dy.double() * xh).abs().sum(0)
        _within(dw, want, U[torch.float32] * want.abs() + (rows * 2.0 ** -24 + F32) * size, "dweight")


def test_rms_norm_repeats_and_streams(layers):
    """The same bits on every call, and on another stream than the tensors were made on."""
    x, r, w = (_rand(i, 3000, 256, dtype=torch.bfloat16) for i in (1, 2, 3))
    w = w[0].contiguous()
    first = (*layers.rms_norm(x, w, r), *layers.rms_norm_backward(x, r, w, x))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = (*layers.rms_norm(x, w, r), *layers.rms_norm_backward(x, r, w, x))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_rms_norm_gradient_against_differences(layers):
    x, r, w = _rand(1, 40, 96), _rand(2, 40, 96), 1 + 0.1 * _rand(3, 96)
    c, e = _rand(4, 40, 96), _rand(5, 40, 96)

    def loss(x, r, w):
        y, s = layers.rms_norm(x, w, r)
        return ((y.double() * c.double()).sum() + (s.double() * e.double()).sum())

    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    y, s = layers.rms_norm(leaves[0], leaves[2], leaves[1])
    ((y * c).sum() + (s * e).sum()).backward()
    h = 1e-2
    for k, base in enumerate((x, r, w)):
        v = _rand(10 + k, *base.shape)
        args = [x, r, w]
        up, down = list(args), list(args)
        up[k], down[k] = base + h * v, base - h * v
        diff = float(loss(*up) - loss(*down)) / (2 * h)
        got = float((leaves[k].grad.double() * v.double()).sum())
        # third-order term h^2 and float32 rounding of 3,840 values over 2 h
        scale = float((leaves[k].grad.double() * v.double()).abs().sum())
        assert abs(diff - got) <= 2e-3 * scale, (k, diff, got)


# ----------------------------------------------------------------------- 8 bits
def _codes(seed, rows, k):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-127, 128, (rows, k), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)


INT8_SIZES = [(1, 1, 1), (1, 50, 900), (12, 70, 1004), (40, 33, 516), (1, 64, 64), (1, 1531, 4096), (2, 33, 17),
              (3, 100, 1000), (5, 513, 129), (8, 256, 2048), (16, 64, 16384), (4, 40, 32757), (60, 24, 8188),
              (9, 128, 128), (16, 136, 96), (17, 250, 384), (31, 1000, 1000), (33, 64, 8192), (64, 512, 512),
              (100, 128, 4097), (127, 129, 255), (128, 256, 256), (129, 257, 300), (333, 1531, 1000),
              (1000, 72, 2048), (2500, 700, 130), (257, 1, 1), (300, 129, 127),
              (600, 256, 4096), (257, 64, 64), (512, 2100, 3200)]


@pytest.mark.parametrize("rows, n, k", INT8_SIZES)
def test_int8_linear(layers, rows, n, k):
    a, b = _codes(1, rows, k), _codes(2, n, k)
    sa, sb = _rand(3, rows).abs() + 0.1, _rand(4, n).abs() + 0.1
    whole = a.double() @ b.double().t()  # below 2^53: exact
    for dtype, bias in ((torch.float32, None), (torch.bfloat16, _rand(5, n) * 100), (torch.float16, None)):
        f = 1e-4 if dtype == torch.float16 else 1.0
        y = layers.int8_linear(a, sa * f, b, sb, bias, out_dtype=dtype)
        prod = whole * (sa * f).double()[:, None] * sb.double()[None, :]
        ref = prod if bias is None else prod + bias.double()
        size = prod.abs() + (0 if bias is None else bias.double().abs())
        _within(y, ref, U[dtype] * ref.abs() + 4 * 2.0 ** -24 * size + TINY[dtype], f"y {dtype}")


def test_int8_linear_extremes(layers):
    """The longest sum of the largest products, and channels of scale 0, infinity and NaN."""
    k = 131071
    a = torch.full((2, k), -128, dtype=torch.int8, device="cuda")
    b = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    b[1] = 127
    one = torch.ones(3, device="cuda")
    y = layers.int8_linear(a, one[:2], b, one, out_dtype=torch.float32)
    for c, v in ((0, 16384.0 * k), (1, -16256.0 * k), (2, 16384.0 * k)):
        assert bool((y[:, c] == torch.tensor(v, dtype=torch.float64).float().cuda()).all())
    sb = torch.tensor([0.0, float("inf"), float("nan")], device="cuda")
    y = layers.int8_linear(a, one[:2], b, sb, out_dtype=torch.float32)
    assert bool((y[:, 0] == 0).all()) and bool(torch.isinf(y[:, 1]).all()) and bool(torch.isnan(y[:, 2]).all())


def test_int8_linear_layouts(layers):
    """Unaligned views and broadcast rows give what their copies give, bit for bit."""
    wa, wb = _codes(1, 280, 600), _codes(2, 90, 600)
    sa, sb = torch.rand(280, device="cuda"), torch.rand(90, device="cuda")
    for rows in (1, 5, 30, 70, 280):
        for a, b in ((wa[:rows, 1:513], wb[:, 7:519]), (wa[:rows, :512], wb[:, 16:528]), (wa[:rows, 3:500], wb[:, 3:500]),
                     (wa[:1, :512].expand(rows, 512), wb[:, :512]), (wa[:rows, :512], wb[:1, :512].expand(90, 512))):
            y = layers.int8_linear(a, sa[:rows], b, sb, out_dtype=torch.float32)
            y2 = layers.int8_linear(a.contiguous(), sa[:rows], b.contiguous(), sb, out_dtype=torch.float32)
            ref = (a.double() @ b.double().t()) * sa[:rows].double()[:, None] * sb.double()
            _within(y, ref, 8 * 2.0 ** -24 * ref.abs(), "y of a view")
            assert torch.equal(y, y2)
    y = layers.int8_linear(wa[:0], sa[:0], wb, sb)
    assert y.shape == (0, 90)
    y = layers.int8_linear(wa[:70].view(7, 10, 600), sa[:70], wb, sb, out_dtype=torch.float32)
    assert y.shape == (7, 10, 90)


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("rows, hidden", [(1, 1), (1, 5632), (3, 7), (4, 256), (9, 512), (5, 513), (2, 8192), (3, 1003),
                                          (2, 16392), (2, 32768), (1, 32767), (700, 1024),
                                          (40, 100), (37, 63), (5, 2051), (9, 2056), (3, 16383), (6, 1030)])
def test_gate_int8(layers, rows, hidden, dtype):
    gu = _rand(1, rows, 2 * hidden, dtype=dtype, scale=3.0)
    codes, scales = layers.gate_int8(gu)
    g, u = gu.double().chunk(2, 1)
    _check_codes(codes, scales, g / (1 + torch.exp(-g)) * u)


def test_gate_int8_special_rows(layers):
    gu = _rand(1, 6, 2 * 320, dtype=torch.bfloat16)
    gu[1] = 0
    gu[2, 10] = float("nan")
    gu[3, 330] = float("inf")
    gu[4, :320] = -100.0  # silu underflows to (almost) nothing
    gu[5, :320] = 1e4     # silu(g) = g
    codes, scales = layers.gate_int8(gu)
    assert float(scales[1]) == 0 and bool((codes[1] == 0).all())
    assert bool(torch.isnan(scales[2:4]).all()) and bool((codes[2:4] == 0).all())
    assert 0 <= float(scales[4]) < 1e-38
    ref = 1e4 * gu[5, 320:].double()
    _within(codes[5].double() * scales[5].double(), torch.where(ref == ref, 9984.0 * gu[5, 320:].double(), ref),
            float(scales[5]) * 0.51, "large gates")
    view = _rand(2, 5, 900, dtype=torch.float16)[:, 5:645]
    c1, s1 = layers.gate_int8(view)
    c2, s2 = layers.gate_int8(view.contiguous())
    assert torch.equal(c1, c2) and torch.equal(s1, s2)
    assert layers.gate_int8(gu[:0])[0].shape == (0, 320)


def test_quantize_weight(layers):
    w = _rand(1, 50, 333, dtype=torch.bfloat16)
    w[7] = 0
    codes, scales = layers.quantize_weight(w)
    assert codes.stride(0) % 16 == 0 and float(scales[7]) == 0
    _check_codes(codes, scales, w.double())


# ----------------------------------------------------------------- feed-forward
def _ffn_inputs(rows, width, hidden, dtype):
    x = _rand(1, rows, width, dtype=dtype)
    wg, wu = (_rand(k, hidden, width, dtype=dtype, scale=width ** -0.5) for k in (2, 3))
    return x, wg, wu, _rand(4, width, hidden, dtype=dtype, scale=hidden ** -0.5), _rand(5, rows, width, dtype=dtype)


def _ffn_ref(x, wg, wu, wd, dy, dtype):
    """The formulas in float64 and, for each result, how far the kernels may be off."""
    u_t, x, wg, wu, wd, dy = U[dtype], *(t.double() for t in (x, wg, wu, wd, dy))
    rows, width = x.shape
    hidden = wg.shape[0]
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = (width * ACC * (x.abs() @ w.abs().t()) for w in (wg, wu))
    sg = 1 / (1 + torch.exp(-g))
    act, slope = g * sg, sg * (1 + g * (1 - sg))
    h = act * u
    few = 16 * 2.0 ** -24  # the activation's own float32 arithmetic
    eh = 1.1 * eg * u.abs() + act.abs() * eu + (u_t + few) * h.abs() + TINY[dtype]  # |silu'| <= 1.1
    y = h @ wd.t()
    ey = u_t * y.abs() + eh @ wd.abs().t() + hidden * ACC * (h.abs() @ wd.abs().t()) + TINY[dtype]
    dh = dy @ wd
    edh = width * ACC * (dy.abs() @ wd.abs())
    du, dg = dh * act, dh * u * slope
    edu = act.abs() * edh + 1.1 * dh.abs() * eg + (u_t + few) * du.abs() + TINY[dtype]
    edg = ((u * slope).abs() * edh + 1.1 * dh.abs() * eu + 0.5 * (dh * u).abs() * eg  # |silu''| <= 0.5
           + u_t * dg.abs() + few * (dh * u).abs() + TINY[dtype])
    dx = dg @ wg + du @ wu
    edx = u_t * dx.abs() + edg @ wg.abs() + edu @ wu.abs() + \
        2 * hidden * ACC * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()) + TINY[dtype]
    out = {"y": (y, ey), "dx": (dx, edx)}
    for name, p, ep, q in (("dw_gate", dg, edg, x), ("dw_up", du, edu, x), ("dw_down", h, eh, dy)):
        v = p.t() @ q
        e = u_t * v.abs() + ep.t() @ q.abs() + rows * ACC * (p.abs().t() @ q.abs()) + TINY[dtype]
        out[name] = (v.t(), e.t()) if name == "dw_down" else (v, e)
    return out


FFN_SIZES = [(1, 1, 1), (1, 70, 150), (3, 1498, 856), (20, 90, 202), (1, 64, 64), (1, 128, 512), (2, 33, 70),
             (3, 128, 300), (4, 256, 1024), (5, 7, 3), (8, 520, 1368), (9, 256, 256), (16, 64, 8192), (6, 40, 8190),
             (50, 24, 6147), (17, 100, 333), (33, 128, 512), (64, 64, 4096), (100, 136, 200), (128, 128, 128),
             (129, 130, 131), (192, 256, 1024), (257, 264, 520), (777, 520, 1368), (3000, 256, 512), (5, 1024, 72),
             (40, 1024, 200), (260, 64, 96), (400, 100, 90), (300, 72, 4100), (257, 1, 1), (333, 1032, 260),
             (300, 2048, 131)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows, width, hidden", FFN_SIZES)
def test_feed_forward_and_gradients(layers, rows, width, hidden, dtype):
    x, wg, wu, wd, dy = _ffn_inputs(rows, width, hidden, dtype)
    ref = _ffn_ref(x, wg, wu, wd, dy, dtype)
    y, saved = layers.feed_forward_train(x, wg, wu, wd)
    assert torch.equal(y, layers.feed_forward(x, wg, wu, wd))
    got = dict(zip(("dx", "dw_gate", "dw_up", "dw_down"), layers.feed_forward_backward(dy, saved)), y=y)
    for name, (want, bound) in ref.items():
        _within(got[name], want, bound, name)
        if want.numel() >= 1000:
            off = float((got[name].double() - want).norm() / want.norm())
            assert off <= 2 * U[dtype], (name, off)


def test_feed_forward_saved_of_another_call(layers):
    x, wg, wu, wd, dy = _ffn_inputs(300, 1024, 64, torch.bfloat16)
    _, saved = layers.feed_forward_train(x, wg, wu, wd)
    assert saved[5] is not None
    for wrong in (saved[:4] + (saved[4][:299], saved[5]), saved[:5] + (saved[5][:-1],), (x[:8],) + saved[1:]):
        with pytest.raises(ValueError):
            layers.feed_forward_backward(dy[:wrong[0].shape[0]], wrong)
    # without the kept projections they are computed again: the same gradients within their roundings
    for a, b in zip(layers.feed_forward_backward(dy, saved), layers.feed_forward_backward(dy, saved[:5] + (None,))):
        off = float((a.double() - b.double()).norm() / a.double().norm())
        assert off <= 2 * U[torch.bfloat16], off


def test_feed_forward_layouts(layers):
    """Unaligned and strided views, a broadcast row, leading dimensions, no rows."""
    dtype = torch.float16
    big, dbig = _rand(1, 600, 200, dtype=dtype), _rand(6, 600, 200, dtype=dtype)
    wgb, wub, wdb = (_rand(k, 300, 400, dtype=dtype, scale=0.1) for k in (2, 3, 4))
    for sl_x, sl_w in ((slice(0, 136), slice(0, 136)), (slice(1, 137), slice(5, 141)), (slice(3, 134), slice(8, 139))):
        width = sl_x.stop - sl_x.start
        for x, dy in ((big[:300, sl_x], dbig[:300, sl_x]), (big[::2, sl_x], dbig[300:, sl_x]),
                      (big[:150, sl_x], dbig[:150, sl_x]), (big[:1, sl_x].expand(270, width), dbig[:270, sl_x]),
                      (big[:1, sl_x].expand(40, width), dbig[:40, sl_x]), (big[:3, sl_x], dbig[:3, sl_x])):
            wg, wu, wd = wgb[:200, sl_w], wub[100:300, sl_w], wdb[:width, 7:207]
            ref = _ffn_ref(x, wg, wu, wd, dy, dtype)
            y, saved = layers.feed_forward_train(x, wg, wu, wd)
            got = dict(zip(("dx", "dw_gate", "dw_up", "dw_down"), layers.feed_forward_backward(dy, saved)), y=y)
            for name, (want, bound) in ref.items():
                _within(got[name], want, bound, f"{name} {sl_x} {tuple(x.stride())}")
    x, wg, wu, wd, dy = _ffn_inputs(12, 64, 96, dtype)
    y = layers.feed_forward(x.view(3, 4, 64), wg, wu, wd)
    assert y.shape == (3, 4, 64) and torch.equal(y.view(12, 64), layers.feed_forward(x, wg, wu, wd))
    y, saved = layers.feed_forward_train(x[:0], wg, wu, wd)
    grads = layers.feed_forward_backward(dy[:0], saved)
    assert y.shape == (0, 64) and grads[0].shape == (0, 64) and all(bool((g == 0).all()) for g in grads[1:])


@pytest.mark.parametrize("rows", [2, 20, 150, 300])
def test_feed_forward_non_finite_rows_stay_apart(layers, rows):
    x, wg, wu, wd, _ = _ffn_inputs(rows, 96, 160, torch.bfloat16)
    clean = layers.feed_forward(x, wg, wu, wd)
    x[1, 5] = float("nan")
    y = layers.feed_forward(x, wg, wu, wd)
    assert bool(torch.isnan(y[1]).all())
    rest = torch.arange(rows, device="cuda") != 1
    assert torch.equal(y[rest], clean[rest])


def test_feed_forward_repeats_streams_and_graphs(layers):
    for rows in (1, 6, 40, 260, 700):
        x, wg, wu, wd, dy = _ffn_inputs(rows, 256, 1024, torch.bfloat16)

        def step():
            y, saved = layers.feed_forward_train(x, wg, wu, wd)
            return (y, *layers.feed_forward_backward(dy, saved))

        first = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            second = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(first, second))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            third = step()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(first, third))


def test_feed_forward_gradient_against_differences(layers):
    dtype = torch.float16
    x, wg, wu, wd, c = _ffn_inputs(60, 64, 96, dtype)
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, wd)]
    layers.feed_forward(*leaves).mul(c).sum().backward()
    h = 0.03
    for k in range(4):
        base = (x, wg, wu, wd)[k]
        v = _rand(20 + k, *base.shape, dtype=dtype, scale=1.0 if k == 0 else base.shape[1] ** -0.5)
        up, down = [x, wg, wu, wd], [x, wg, wu, wd]
        up[k], down[k] = base + h * v, base - h * v
        step = up[k].double() - down[k].double()  # the step as float16 has it
        diff = float(((layers.feed_forward(*up).double() - layers.feed_forward(*down).double()) * c.double()).sum())
        got = float((leaves[k].grad.double() * step).sum())
        # rounding of 2 x 3,840 outputs of size <= 4 to float16 adds in quadrature; h^2 truncation below 1 %
        noise = 4 * U[dtype] * float(c.double().norm()) * 2
        assert abs(diff - got) <= noise + 0.02 * abs(got) + 0.02 * float((leaves[k].grad.double() * step).norm()), (k, diff, got)


# ------------------------------------------------------------------ the sublayer
def test_blocks_train_and_serve(layers):
    torch.manual_seed(0)
    block = layers.FeedForwardBlock(256, 1024)
    x, r, target = (_rand(k, 192, 256, dtype=torch.bfloat16) for k in (1, 2, 3))
    opt = torch.optim.SGD(block.parameters(), lr=10.0)
    losses = []
    for _ in range(6):
        opt.zero_grad()
        out, s = block(x, r)
        loss = ((out + s).float() - target.float()).square().mean()
        loss.backward()
        assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in block.parameters())
        opt.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < losses[0]
    with torch.no_grad():
        out, s = block(x, r)
        served, s8 = layers.Int8FeedForwardBlock(block)(x, r)
    assert torch.equal(s, s8)
    # three roundings to 8 bits of about 1 part in 36 sqrt(12) of a row's rms each
    off = float((served.double() - out.double()).norm() / out.double().norm())
    assert off <= 4 * 3 ** 0.5 / (36 * 12 ** 0.5), off


def test_autograd_hands_over_any_gradient(layers):
    """Broadcast and transposed gradients, an output that nothing reads, leading dimensions."""
    x, r = _rand(1, 2, 9, 64, dtype=torch.bfloat16), _rand(2, 2, 9, 64, dtype=torch.bfloat16)
    w = torch.ones(64, device="cuda", requires_grad=True)
    for use in (lambda y, s: y.sum(), lambda y, s: s.sum(), lambda y, s: (y.transpose(1, 2) * 2).sum() + s.sum()):
        leaf, other = x.clone().requires_grad_(), r.clone().requires_grad_()
        w.grad = None
        use(*layers.rms_norm(leaf, w, other)).backward()
        xd, rd, wd = x.float().requires_grad_(), r.float().requires_grad_(), w.detach().clone().requires_grad_()
        s = ((xd + rd).bfloat16().float() - (xd + rd)).detach() + (xd + rd)  # rounded, with the sum's gradient
        y = s * torch.rsqrt(s.square().mean(-1, keepdim=True) + 1e-6) * wd
        use(y, s).backward()
        assert torch.equal(leaf.grad, other.grad)
        _within(leaf.grad, xd.grad.double(), 2 * U[torch.bfloat16] * (xd.grad.double().abs() + 0.1), "dx")
        if wd.grad is not None and bool((wd.grad != 0).any()):
            _within(w.grad, wd.grad.double(), 1e-3 * (1 + wd.grad.double().abs()), "dweight")
    ws = [t.requires_grad_() for t in _ffn_inputs(18, 64, 96, torch.bfloat16)[1:4]]
    leaf = x.clone().requires_grad_()
    layers.feed_forward(leaf, *ws).sum().backward()
    _, saved = layers.feed_forward_train(x.view(18, 64), *(t.detach() for t in ws))
    grads = layers.feed_forward_backward(torch.ones(18, 64, device="cuda", dtype=torch.bfloat16), saved)
    for got, want in zip((leaf.grad.view(18, 64), *(t.grad for t in ws)), grads):
        assert torch.equal(got, want)


# --------------------------------------------------------------------- refusals
def test_refusals(layers):
    from so3lr_b200 import So3lrError
    x = _rand(1, 4, 64, dtype=torch.bfloat16)
    w = torch.ones(64, device="cuda")
    for call in (
        lambda: layers.rms_norm(x.cpu(), w.cpu()),
        lambda: layers.rms_norm(x, w[:63]),
        lambda: layers.rms_norm(x, w.half()),
        lambda: layers.rms_norm(x, w, x[:3]),
        lambda: layers.rms_norm(x, w, x.float()),
        lambda: layers.rms_norm(x.double(), w),
        lambda: layers.rms_norm(x.t(), torch.ones(4, device="cuda")),
        lambda: layers.rms_norm(_rand(1, 6, 4, 64).transpose(0, 1)[:, :, :32], w[:32]),
        lambda: layers.rms_norm_backward(x[:3], x, w),
        lambda: layers.gate_int8(x[:, :63]),
        lambda: layers.int8_linear(x, w[:4], x, w[:4]),
        lambda: layers.int8_linear(x.to(torch.int8), w[:3], x.to(torch.int8), w[:4]),
        lambda: layers.int8_linear(x.to(torch.int8), w[:4], x.to(torch.int8)[:, :32], w[:4]),
        lambda: layers.int8_linear(x.to(torch.int8), w[:4], x.to(torch.int8), w[:4], out_dtype=torch.int32),
        lambda: layers.dequantize_int8(x.to(torch.int8), w[:3]),
        lambda: layers.feed_forward(x, x, x, x),
        lambda: layers.feed_forward(x, x, x[:3], x.t().contiguous()),
        lambda: layers.feed_forward(x.float(), x.float(), x.float(), x.float().t().contiguous()),
        lambda: layers.feed_forward(x, x.half(), x, x.t().contiguous()),
        lambda: layers.feed_forward(x, x, x, x.t()),
    ):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(So3lrError, match="width must be in 1..16384"):
        layers.rms_norm(_rand(1, 1, 16385), torch.ones(16385, device="cuda"))
    with pytest.raises(So3lrError, match="hidden must be in 1..32768"):
        layers.gate_int8(_rand(1, 1, 65538))
    with pytest.raises(So3lrError, match="k must be in 1..131071"):
        layers.int8_linear(torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), w[:1],
                           torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), w[:1])
    with pytest.raises(So3lrError, match="eps"):
        layers.rms_norm(x, w, eps=-1.0)


# ------------------------------------------------------------- past 32-bit offsets
@pytest.mark.parametrize("off_boundary", [0, 1])
@pytest.mark.parametrize("rows", [9, 300])
def test_inputs_past_32_bit_offsets(layers, rows, off_boundary):
    """Rows spread over more than 2^31 elements give what the same rows side by side give."""
    stride = ((2 ** 31 + 2 ** 20) // (rows - 1) + 7) // 8 * 8 + off_boundary
    big = torch.empty((rows - 1) * stride + 512, device="cuda", dtype=torch.bfloat16)

    def spread(t):
        view = big.as_strided(t.shape, (stride, 1))
        view.copy_(t)
        return view

    x, w = _rand(1, rows, 256, dtype=torch.bfloat16), 1 + 0.1 * _rand(2, 256)
    dy = _rand(3, rows, 256, dtype=torch.bfloat16)
    y, s = layers.rms_norm(spread(x), w, dy)
    _within(s, (x.float() + dy.float()).to(torch.bfloat16).double(), 0.0, "s")
    ref, _ = _norm_ref(s.double(), w.double())
    _within(y, ref, (U[torch.bfloat16] + F32) * ref.abs() + TINY[torch.bfloat16], "y")
    dx, dw = layers.rms_norm_backward(dy, spread(x), w)
    dx2, dw2 = layers.rms_norm_backward(dy, x, w)
    _within(dx, dx2.double(), 2 * U[torch.bfloat16] * (dx2.double().abs() + 1e-3), "dx")
    _within(dw, dw2.double(), 1e-4 * dw2.double().abs().max(), "dweight")
    gate, _ = layers.gate_int8(spread(x))
    assert torch.equal(gate, layers.gate_int8(x)[0])
    wg, wu, wd = (_rand(i, *n, dtype=torch.bfloat16, scale=0.06) for i, n in ((4, (300, 256)), (5, (300, 256)), (6, (256, 300))))
    assert torch.equal(layers.feed_forward(spread(x), wg, wu, wd), layers.feed_forward(x, wg, wu, wd))
    _, saved = layers.feed_forward_train(spread(x), wg, wu, wd)
    got = layers.feed_forward_backward(dy, saved)
    _, saved = layers.feed_forward_train(x, wg, wu, wd)
    assert all(torch.equal(a, b) for a, b in zip(got, layers.feed_forward_backward(dy, saved)))
    b = _codes(7, 300, 512)
    sa, sb = torch.ones(rows, device="cuda"), torch.ones(300, device="cuda")
    a = _codes(8, rows, 512)
    far = big.view(torch.int8).as_strided((rows, 512), (2 * stride, 1))
    far.copy_(a)
    want = layers.int8_linear(a, sa, b, sb, out_dtype=torch.float32)
    assert torch.equal(layers.int8_linear(far, sa, b, sb, out_dtype=torch.float32), want)
    assert torch.equal(layers.int8_linear(b, sb, far, sa, out_dtype=torch.float32), want.T)


def test_results_past_32_bit_offsets(layers):
    rows, width = 2 ** 31 // 4096 + 5, 4096
    codes, scales = _codes(1, rows, width), 0.01 + torch.rand(rows, device="cuda")
    x = layers.dequantize_int8(codes, scales)
    for part in (slice(0, 3), slice(rows - 5, rows)):
        assert torch.equal(x[part], (codes[part].float() * scales[part, None]).bfloat16())
    w = 1 + 0.1 * _rand(2, width)
    codes, scales, _ = layers.rms_norm_int8(x, w, eps=EPS)
    ref, _ = _norm_ref(x[-5:].double(), w.double())
    _check_codes(codes[-5:], scales[-5:], ref)
    del codes
    y, _ = layers.rms_norm(x, w, eps=EPS)
    _within(y[-5:], ref, (U[torch.bfloat16] + F32) * ref.abs() + TINY[torch.bfloat16], "y")
    del x, y
    rows, n, k = 70001, 32768, 32
    a, b = _codes(3, rows, k), _codes(4, n, k)
    y = layers.int8_linear(a, torch.ones(rows, device="cuda"), b, torch.ones(n, device="cuda"))
    want = (a[-40:].double() @ b.double().T).bfloat16()  # sums below 2^24: exact in float32
    assert torch.equal(y[-40:], want)
