"""AdamW steps (so3lr_b200.optim) on the GPU, against the plain formula in float64.

u is float32's unit roundoff, 2^-24. One step from a given state: with
S = b1 |m| + (1 - b1) |g| the new m is within 4 u S (each constant, product and sum rounded
once), v within 5 u of itself. The update lr / bc1 m / (sqrt(v / bc2) + eps) carries m's
error, half of v's, 4 u of the root, 4 u of the division, the coefficients' and the
products' roundings: 32 u of the update with S in m's place. p adds 5 u |p|, a 16-bit p
without a master its own rounding.

8-bit moments: decoding adds at most 12 u to what the formula is given (t, its powers, the
scale). A code c must be the nearest: the new moment lies between the values of the codes
|c| - 1/2 and |c| + 1/2, the code's own arithmetic (reciprocal, roots, product) counted as
32 u of 127 or 255, the moment's error as 16 u S for m and 20 u v for v.
"""
import copy

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U32 = 2.0 ** -24
U = {torch.float32: U32, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


@pytest.fixture(scope="module")
def optim():
    from so3lr_b200 import optim
    return optim


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _values(codes, scales):
    """An 8-bit moment in float64, and its scale for each element"""
    n = codes.numel()
    top = scales.double().repeat_interleave(256)[:n].view(codes.shape)
    c = codes.double()
    return (c * c.abs() / 127 ** 2 if codes.dtype == torch.int8 else (c / 255) ** 4) * top, top


def _make(optim, shapes, dtype, grad_dtype=None, eight=(), master=True, seed=0):
    """A state well into a run: params, grads, moments (8 bits for the indices in `eight`), counters, masters."""
    g = _gen(seed)
    s = dict(p=[], g=[], m=[], v=[], ms=[], vs=[], master=[])
    for i, shape in enumerate(shapes):
        x = torch.randn(shape, generator=g, device="cuda")
        n, blocks = x.numel(), (x.numel() + 255) // 256
        s["p"].append(x.to(dtype))
        s["master"].append(x.clone() if master and dtype != torch.float32 else None)
        s["g"].append((torch.randn(shape, generator=g, device="cuda") * 1e-2).to(grad_dtype or dtype))
        if i in eight:
            s["m"].append(torch.randint(-127, 128, (n,), generator=g, device="cuda").to(torch.int8).view(shape))
            s["v"].append(torch.randint(1, 256, (n,), generator=g, device="cuda").to(torch.uint8).view(shape))
            s["ms"].append(torch.rand(blocks, generator=g, device="cuda") * 1e-2 + 1e-4)
            s["vs"].append(torch.rand(blocks, generator=g, device="cuda") * 1e-4 + 1e-6)
        else:
            s["m"].append(torch.randn(shape, generator=g, device="cuda") * 1e-3)
            s["v"].append(torch.rand(shape, generator=g, device="cuda") * 1e-4)
            s["ms"].append(None)
            s["vs"].append(None)
    s["steps"] = torch.randint(0, 50, (len(shapes),), generator=g, device="cuda")
    return s


def _step(optim, s, **more):
    optim.adamw_step(s["p"], s["g"], s["m"], s["v"], s["steps"], exp_avg_scales=s["ms"], exp_avg_sq_scales=s["vs"],
                     masters=s["master"], **{**HYPER, **more})


def _within(got, want, bound, what):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, first at "
                                 f"{bad.nonzero()[0].tolist()}: {float(off[bad][0]):.3e} > {float(bound[bad][0]):.3e}")


def _check_codes(codes, scales, want, err, what):
    """Each code is the nearest to `want`, which may be off by `err`; the scales are the blocks' largest."""
    signed = codes.dtype == torch.int8
    levels, power = (127, 2) if signed else (255, 4)
    n = codes.numel()
    flat = lambda t: torch.nn.functional.pad(t.reshape(-1), (0, -n % 256)).view(-1, 256)  # noqa: E731
    largest = flat(want.abs()).amax(1)
    _within(scales, largest, flat(err).amax(1) + U32 * largest + 2.0 ** -126, what + " scales")
    top = scales.double().repeat_interleave(256)[:n].view(codes.shape)
    c, slack = codes.double(), 32 * U32 * levels
    low = top * (((c.abs() - 0.5 - slack).clamp(min=0)) / levels) ** power
    high = top * ((c.abs() + 0.5 + slack) / levels) ** power
    if not signed:
        low = torch.where(c == 1, torch.zeros_like(low), low)  # what is not zero has code 1 at least
        assert bool(((c >= 1) | (want <= 2.0 ** -149) | (top == 0)).all()), what + ": a value above zero became zero"
    size = want.abs()
    assert bool(((size >= low - err) & (size <= high + err)).all()), what + ": a code is not the nearest"
    if signed:
        assert bool(((c == 0) | (c.sign() == want.sign()) | (size <= err)).all()), what + ": sign"


def _check(before, after, hyper=HYPER, what=""):
    b1, b2 = hyper["betas"]
    for i in range(len(before["p"])):
        name = f"{what} tensor {i}"
        t = int(before["steps"][i]) + 1
        assert int(after["steps"][i]) == t
        dtype = before["p"][i].dtype
        master = before["master"][i]
        p0, g = (before["p"][i] if master is None else master).double(), before["g"][i].double()
        eight = before["ms"][i] is not None
        m0 = _values(before["m"][i], before["ms"][i])[0] if eight else before["m"][i].double()
        v0 = _values(before["v"][i], before["vs"][i])[0] if eight else before["v"][i].double()
        m, v, size = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g, b1 * m0.abs() + (1 - b1) * g.abs()
        scale = hyper["lr"] / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + hyper["eps"])
        p = p0 * (1 - hyper["lr"] * hyper["weight_decay"]) - scale * m
        err = 5 * U32 * p0.abs() + (64 if eight else 32) * U32 * scale * size
        if master is not None:
            _within(after["master"][i], p, err, name + " master")
            assert torch.equal(after["p"][i], after["master"][i].to(dtype)), name + ": not the master's rounding"
        else:
            _within(after["p"][i], p, err + (U[dtype] * (p.abs() + err) + TINY[dtype] if dtype != torch.float32 else 0), name)
        if eight:
            _check_codes(after["m"][i], after["ms"][i], m, 16 * U32 * size, name + " m")
            _check_codes(after["v"][i], after["vs"][i], v, 20 * U32 * v, name + " v")
        else:
            _within(after["m"][i], m, 4 * U32 * size, name + " m")
            _within(after["v"][i], v, 5 * U32 * v + 2.0 ** -149, name + " v")


LENGTHS = [(1,), (7,), (8,), (255,), (256,), (257,), (31, 67), (2048,), (2049,), (0,), (64, 130), (100003,)]


@pytest.mark.parametrize("master", [True, False])
@pytest.mark.parametrize("dtype, grad_dtype", [(torch.float32, None), (torch.bfloat16, None), (torch.float16, None),
                                               (torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
def test_step(optim, dtype, grad_dtype, master):
    s = _make(optim, LENGTHS + LENGTHS, dtype, grad_dtype, eight=range(len(LENGTHS)), master=master)
    before = copy.deepcopy(s)
    _step(optim, s)
    _check(before, s)
    for a, b in zip(before["g"], s["g"]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("count", [1, 23, 24, 25, 399, 400, 401, 900])
def test_number_of_tensors(optim, count):
    """One launch or several, and all counters."""
    shapes = [(1 + 37 * i % 3001,) for i in range(count)]
    s = _make(optim, shapes, torch.bfloat16, eight=range(0, count, 3))
    before = copy.deepcopy(s)
    _step(optim, s)
    _check(before, s)


@pytest.mark.parametrize("shift", [1, 2, 4])
def test_views_off_the_boundaries(optim, shift):
    """Tensors that start on any element, and what lies around them."""
    n, pad = 5000, 16
    whole = dict(p=torch.bfloat16, g=torch.bfloat16, m=torch.int8, v=torch.uint8, master=torch.float32, ms=torch.float32,
                 vs=torch.float32)
    s = _make(optim, [(n,)], torch.bfloat16, eight=[0])
    buffers = {}
    for k, dtype in whole.items():
        t = s[k][0]
        buffers[k] = torch.full((t.numel() + 2 * pad,), 77, device="cuda").to(dtype)
        s[k] = [buffers[k][shift:shift + t.numel()].copy_(t)]
    before = copy.deepcopy(s)
    _step(optim, s)
    _check(before, s)
    for k, b in buffers.items():
        size = s[k][0].numel()
        assert bool((b[:shift] == 77).all()) and bool((b[shift + size:] == 77).all()), k


def test_hyperparameters(optim):
    for more in (dict(lr=0.0), dict(betas=(0.0, 0.0)), dict(weight_decay=0.0), dict(eps=1e-3), dict(lr=1.0, betas=(0.5, 0.999))):
        s = _make(optim, [(300,), (257,)], torch.float32, eight=[1])
        before = copy.deepcopy(s)
        _step(optim, s, **more)
        _check(before, s, {**HYPER, **more}, str(more))


def test_first_steps_from_zero(optim):
    """Zero codes and scales are zero moments; the corrections of t = 1, 2 lose no digits."""
    s = _make(optim, [(1000,), (1000,)], torch.float32, eight=[1])
    for k in ("m", "v"):
        for t in s[k] + [s[k + "s"][1]]:
            t.zero_()
    s["steps"].zero_()
    hyper = dict(HYPER, betas=(0.9, 0.999))
    for k in range(3):
        before = copy.deepcopy(s)
        _step(optim, s, betas=(0.9, 0.999))
        _check(before, s, hyper, f"step {k + 1}")


def test_far_steps(optim):
    s = _make(optim, [(100,)], torch.float32)
    s["steps"].fill_((1 << 40) + 3)
    before = copy.deepcopy(s)
    _step(optim, s)
    _check(before, s)


def test_not_finite(optim):
    """Float32 moments carry an infinity or a NaN where it is; 8-bit ones in the 256 of its scale."""
    for bad in (float("inf"), float("-inf"), float("nan")):
        s = _make(optim, [(1000,), (1000,)], torch.float32, eight=[1])
        for g in s["g"]:
            g[300] = bad
        before = copy.deepcopy(s)
        _step(optim, s)
        assert not bool(torch.isfinite(s["p"][0][300])) and not bool(torch.isfinite(s["m"][0][300]))
        fine = torch.arange(1000, device="cuda") != 300
        for k in ("p", "m", "v"):
            assert bool(torch.isfinite(s[k][0][fine]).all())
        assert torch.isnan(s["ms"][1]).tolist() == torch.isnan(s["vs"][1]).tolist() == [False, True, False, False]
        assert bool((s["m"][1][256:512] == 0).all()) and bool((s["v"][1][256:512] == 0).all())
        assert torch.isnan(optim.moment_values(s["m"][1], s["ms"][1])).nonzero().flatten().tolist() == list(range(256, 512))
        assert bool(torch.isfinite(s["p"][1][fine]).all())
        _step(optim, s)
        assert bool(torch.isnan(s["p"][1][256:512]).all()) and bool(torch.isfinite(s["p"][1][:256]).all())


def test_small_and_large_moments(optim):
    """Scales at the ends of float32: below its normal numbers they are zero."""
    n = 512
    for scale in (1e-25, 1e-22, 1e-19, 1e-16, 1e-10, 1e10, 1e18):
        s = _make(optim, [(n,)], torch.float32, eight=[0])
        for k in ("m", "v", "ms", "vs"):
            s[k][0].zero_()
        s["g"][0].copy_(torch.randn(n, generator=_gen(3), device="cuda") * scale)
        before = copy.deepcopy(s)
        _step(optim, s)
        want = (1 - HYPER["betas"][1]) * before["g"][0].double() ** 2
        live = want.view(2, 256).amax(1) >= 2.0 ** -125
        dead = want.view(2, 256).amax(1) < 2.0 ** -127
        assert bool((s["vs"][0][live] > 0).all()) and bool((s["vs"][0][dead] == 0).all())
        if bool(live.all()):
            _check_codes(s["v"][0], s["vs"][0], want, 20 * U32 * want + 2.0 ** -149, "v")
        assert bool(torch.isfinite(s["p"][0]).all())


@pytest.mark.parametrize("n", [1, 255, 256, 257, 4096, 100003])
def test_moment_values(optim, n):
    codes = torch.randint(-127, 128, (n,), generator=_gen(1), device="cuda").to(torch.int8)
    scales = torch.rand((n + 255) // 256, generator=_gen(2), device="cuda") + 0.5
    for c in (codes, torch.randint(0, 256, (n,), generator=_gen(3), device="cuda").to(torch.uint8)):
        want, _ = _values(c, scales)
        for dtype in U:
            got = optim.moment_values(c, scales, dtype)
            assert got.dtype == dtype and got.shape == c.shape
            _within(got, want, (U[dtype] + 12 * U32) * want.abs() + TINY[dtype], str(dtype))
    # the largest of a block is kept exactly
    assert torch.equal(optim.moment_values(torch.full((n,), -127, dtype=torch.int8, device="cuda"), scales),
                       -scales.repeat_interleave(256)[:n])
    assert torch.equal(optim.moment_values(torch.full((n,), 255, dtype=torch.uint8, device="cuda"), scales),
                       scales.repeat_interleave(256)[:n])


def test_captured_and_replayed(optim):
    """A graph counts its own steps, reads the rate from the GPU, and does what the same calls do."""
    shapes = [(513,), (2048, 9), (70,)]
    lr = torch.full((), 3e-3, device="cuda")
    eager, graphed = (_make(optim, shapes, torch.bfloat16, eight=[1]) for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    keep = copy.deepcopy(graphed)
    with torch.cuda.graph(graph):
        _step(optim, graphed, lr=lr)
    for a, b in zip(keep["p"], graphed["p"]):
        assert torch.equal(a, b)
    for k in range(3):
        lr.fill_(3e-3 / (k + 1))
        for a, b in zip(eager["g"], graphed["g"]):
            b.copy_(a.mul_(-0.7))
        _step(optim, eager, lr=lr)
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(eager["steps"], graphed["steps"])
    for k in ("p", "master", "m", "v", "ms", "vs"):
        for a, b in zip(eager[k], graphed[k]):
            assert a is None or torch.equal(a, b), k


def test_two_streams_at_once(optim):
    made = [_make(optim, [(4097,), (300000,)], torch.bfloat16, eight=[1], seed=k) for k in range(2)]
    before = copy.deepcopy(made)
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    for s, stream in zip(made, streams):
        with torch.cuda.stream(stream):
            _step(optim, s)
    torch.cuda.synchronize()
    for b, s in zip(before, made):
        _check(b, s)


def test_calls_back_to_back(optim):
    """A step reads what the one just before wrote."""
    apart, together = (_make(optim, [(70000,), (33,)], torch.float32, eight=[0]) for _ in range(2))
    for _ in range(5):
        _step(optim, apart)
        torch.cuda.synchronize()
    for _ in range(5):
        _step(optim, together)
    for k in ("p", "m", "v", "ms"):
        for a, b in zip(apart[k], together[k]):
            assert a is None or torch.equal(a, b)


# ------------------------------------------------------------------ the optimiser
def _model(dtype=torch.bfloat16):
    torch.manual_seed(3)
    return torch.nn.Sequential(torch.nn.Linear(70, 131), torch.nn.SiLU(), torch.nn.Linear(131, 41)).to("cuda", dtype)


def _backward(model, seed):
    x = torch.randn(64, 70, generator=_gen(seed), device="cuda").to(next(model.parameters()).dtype)
    model.zero_grad()
    model(x).float().square().mean().backward()


def _state_of(optimizer, params):
    take = lambda key: [optimizer.state[p].get(key) for p in params]  # noqa: E731
    return copy.deepcopy(dict(p=[p.detach() for p in params], g=[p.grad for p in params], m=take("exp_avg"),
                              v=take("exp_avg_sq"), ms=take("exp_avg_scale"), vs=take("exp_avg_sq_scale"),
                              master=take("master"), steps=take("step")))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", list(U))
def test_optimizer(optim, dtype, bits):
    model = _model(dtype)
    params = list(model.parameters())
    adam = optim.AdamW(params, moment_bits=bits, **HYPER)
    for k in range(4):
        _backward(model, k)
        if k == 0:
            for p in params:
                adam._start(p, adam.param_groups[0])
        before = _state_of(adam, params)
        adam.step()
        _check(before, _state_of(adam, params), what=f"step {k}")
    kinds = {adam.state[p]["exp_avg"].dtype for p in params}
    assert kinds == ({torch.float32} if bits == 32 else {torch.float32, torch.int8})
    assert all(("master" in adam.state[p]) == (dtype != torch.float32) for p in params)


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_state_is_saved_and_loaded(optim, bits, tmp_path):
    """A run that is stopped and taken up again goes on with the same bits."""
    model = _model()
    adam = optim.AdamW(model.parameters(), moment_bits=bits, **HYPER)
    for k in range(3):
        _backward(model, k)
        adam.step()
    torch.save(dict(model=model.state_dict(), adam=adam.state_dict()), tmp_path / "run.pt")
    saved = torch.load(tmp_path / "run.pt")
    other = _model()
    other.load_state_dict(saved["model"])
    again = optim.AdamW(other.parameters(), moment_bits=bits, **HYPER)
    again.load_state_dict(saved["adam"])
    for k in range(3, 6):
        for m, a in ((model, adam), (other, again)):
            _backward(m, k)
            a.step()
    for p, q in zip(model.parameters(), other.parameters()):
        assert torch.equal(p, q)
        for key, value in adam.state[p].items():
            assert torch.equal(value, again.state[q][key]) and value.dtype == again.state[q][key].dtype, key


def test_optimizer_groups_schedules_and_missing_gradients(optim):
    model = _model(torch.float32)
    first, second = list(model[0].parameters()), list(model[2].parameters())
    adam = optim.AdamW([dict(params=first), dict(params=second, lr=1e-4, weight_decay=0.0, moment_bits=8)], **HYPER)
    schedule = torch.optim.lr_scheduler.StepLR(adam, 1, gamma=0.5)
    for k in range(3):
        _backward(model, k)
        if k == 1:
            first[0].grad = None
        keep = first[0].detach().clone()
        adam.step()
        schedule.step()
        assert torch.equal(keep, first[0]) == (k == 1)
    assert [int(adam.state[p]["step"]) for p in first + second] == [2, 3, 3, 3]
    assert adam.param_groups[0]["lr"] == HYPER["lr"] / 8
    closure = lambda: model(torch.ones(1, 70, device="cuda")).square().mean()  # noqa: E731
    assert float(adam.step(closure).detach()) > 0


def test_optimizer_rate_on_the_gpu(optim):
    """A rate that is a tensor, and a schedule that writes into it, do what numbers do."""
    runs = []
    for lr in (HYPER["lr"], torch.tensor(HYPER["lr"], device="cuda")):
        model = _model()
        adam = optim.AdamW(model.parameters(), **{**HYPER, "lr": lr})
        schedule = torch.optim.lr_scheduler.StepLR(adam, 1, gamma=0.5)
        for k in range(3):
            _backward(model, k)
            adam.step()
            schedule.step()
        runs.append([adam.state[p]["master"] for p in model.parameters()])
    for a, b in zip(*runs):  # the rate itself is rounded to float32: 2^-24 of three updates of at most 2 lr
        assert bool(((a - b).abs() <= 2.0 ** -23 * (a.abs() + 6 * HYPER["lr"])).all())


def test_optimizer_marks_parameters_as_changed(optim):
    """A backward pass that kept a parameter from before the step is refused, as after torch's own steps."""
    w = torch.nn.Parameter(torch.ones(8, device="cuda"))
    adam = optim.AdamW([w])
    loss = (w * w).sum()
    w.grad = torch.ones_like(w)
    adam.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_transposed_gradients(optim):
    w = torch.nn.Parameter(torch.randn(30, 20, device="cuda"))
    adam = optim.AdamW([w], **HYPER)
    adam._start(w, adam.param_groups[0])
    w.grad = torch.randn(20, 30, device="cuda").t()
    before = _state_of(adam, [w])
    adam.step()
    _check(before, _state_of(adam, [w]))


# -------------------------------------------------------------------- refusals
def test_refusals(optim):
    def refused(match, kind=ValueError, **change):
        s = _make(optim, [(300,), (40,)], torch.bfloat16, eight=[0])
        hyper = {k: change.pop(k) for k in list(change) if k in ("lr", "betas", "eps", "weight_decay")}
        for k, v in change.items():
            s[k] = v(s[k]) if callable(v) else v
        before = copy.deepcopy(s)
        with pytest.raises(kind, match=match):
            _step(optim, s, **hyper)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(before["p"], s["p"])) or "p" in change

    from so3lr_b200 import So3lrError
    f32 = lambda l: [t.float() for t in l]  # noqa: E731
    refused("as many tensors", g=lambda l: l[:1])
    refused("must be a list", g=3)
    refused("must be a tensor", g=[None, None])
    refused("elements", g=lambda l: [t[:-1] for t in l])
    refused("on cpu", g=lambda l: [t.cpu() for t in l])
    refused("no CPU path", p=lambda l: [t.cpu() for t in l])
    refused("must be torch.bfloat16", g=lambda l: [t.half() for t in l])
    refused("params must be one of", p=lambda l: [t.double() for t in l])
    refused("exp_avgs.0. must be torch.int8", m=f32)
    refused("exp_avg_sqs.0. must be torch.uint8", v=f32)
    refused("given together", vs=lambda l: [None, None])
    refused("must have 2 elements", ms=lambda l: [l[0][:1], None])
    refused("must be contiguous", g=lambda l: [l[0].repeat_interleave(2)[::2], l[1]])
    refused("steps must be", steps=lambda t: t.int())
    refused("steps must be", steps=lambda t: t[:1])
    refused("lr must be", lr=torch.zeros(1))
    refused("lr must be a number", lr="fast")
    refused("lr must be finite", kind=So3lrError, lr=float("nan"))
    refused("lr must be finite", kind=So3lrError, lr=-1.0)
    refused("beta1 and beta2", kind=So3lrError, betas=(1.0, 0.9))
    refused("eps must be", kind=So3lrError, eps=0.0)
    refused("weight_decay must be", kind=So3lrError, weight_decay=-0.1)
    refused("parameters overlap", kind=So3lrError, p=lambda l: [l[0], l[0][:40]])
    refused("step counters overlap", kind=So3lrError, steps=lambda t: [t[:1], t[:1]])
    with pytest.raises(So3lrError, match="master is for 16-bit"):
        s = _make(optim, [(300,)], torch.float32)
        s["master"] = [s["p"][0].clone()]
        _step(optim, s)
    with pytest.raises(ValueError, match="codes must be"):
        optim.moment_values(torch.zeros(3, device="cuda"), torch.zeros(1, device="cuda"))
    with pytest.raises(ValueError, match="scales must be"):
        optim.moment_values(torch.zeros(300, dtype=torch.int8, device="cuda"), torch.zeros(1, device="cuda"))
    with pytest.raises(ValueError, match="dense"):
        w = torch.nn.Parameter(torch.ones(4, 4, device="cuda"))
        w.grad = torch.eye(4, device="cuda").to_sparse()
        optim.AdamW([w]).step()
    optim.adamw_step([], [], [], [], [])
