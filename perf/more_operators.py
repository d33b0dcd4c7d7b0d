"""Measured cases of a block's dense layer, its norms and its optimiser
(so3lr_b200.layers, so3lr_b200.optim).

Rows are atoms (or tokens), columns their features. Three operators:

  linear    y = act(x W^T + bias) + residual, forward alone (serving) or forward
            and backward (training)
  sandwich  the norms on both sides of a block's boundary: the block's output is
            normalised, gated and added to the scaled stream, and the stream is
            normalised for the next block:
              s = residual * scale + gate * norm(x) * weight
              y = norm(s) * next_weight
  adamw     one AdamW step over all tensors of a stack of such blocks, moments in
            32 bits or in 8 (matrices; vectors keep 32), 16-bit matrices with
            float32 masters

`run` computes the plain form in 32 bits where `own` is false and calls the
framework where it is true.
"""
import math

import torch

own = False

EPS = 1e-6
LR, BETA1, BETA2, ADAM_EPS, DECAY = 3e-4, 0.9, 0.999, 1e-8, 0.1
BLOCK = 256  # elements of a tensor that share the scale of an 8-bit moment
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# --------------------------------------------------------------------- cases
def listed():
    return [
        # one row through a square layer: the weight's bytes are all there is
        dict(name="linear_one_row", op="linear", mode="serve", rows=1, k=4096, n=4096, dtype="bf16", act="silu",
             bias=True, residual=False),
        # training the first layer of an atom-wise network at the wider shipped model's width on the water box
        dict(name="linear_train_water_box", op="linear", mode="train", rows=24000, k=256, n=1024, dtype="bf16",
             act="silu", bias=True, residual=False),
        # a small batch, ragged in every length
        dict(name="linear_ragged", op="linear", mode="train", rows=333, k=1000, n=1531, dtype="f16", act="gelu",
             bias=True, residual=True),
        # training, the largest: a wide layer on a long batch
        dict(name="linear_train_large", op="linear", mode="train", rows=8192, k=4096, n=8192, dtype="bf16",
             act="gelu_tanh", bias=True, residual=True),
        # one row between two blocks: the call is all latency
        dict(name="sandwich_one_row", op="sandwich", mode="serve", rows=1, width=2048, dtype="bf16", gate=True,
             scale=True),
        # training on the 24,000-atom water box at the wider shipped model's feature width
        dict(name="sandwich_train_water_box", op="sandwich", mode="train", rows=24000, width=256, dtype="bf16",
             gate=True, scale=True),
        # training at a width that no vector load divides
        dict(name="sandwich_train_odd", op="sandwich", mode="train", rows=3001, width=1003, dtype="f32", gate=True,
             scale=False),
        # training, the largest batch
        dict(name="sandwich_train_large", op="sandwich", mode="train", rows=16384, width=4096, dtype="bf16", gate=True,
             scale=True),
        # one block's tensors: few and small, so launches and host time count
        dict(name="adamw_one_block", op="adamw", width=256, hidden=1024, layers=1, dtype="bf16", bits=32),
        # a deep stack of odd widths: hundreds of small tensors, 8-bit moments
        dict(name="adamw_many_odd", op="adamw", width=251, hidden=1003, layers=48, dtype="f16", bits=8),
        # a large stack, moments in 32 bits
        dict(name="adamw_large", op="adamw", width=2048, hidden=8192, layers=4, dtype="bf16", bits=32),
        # the largest, moments in 8 bits
        dict(name="adamw_large_8bit", op="adamw", width=2048, hidden=8192, layers=8, dtype="bf16", bits=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A length between lo and hi, even over its logarithm: one in four as it falls, the others as layers have them."""
    n, step = _log(rng, lo, hi), rng.choice((1, 8, 16, 64))
    return max(lo, min(hi, n // step * step))


def draw(rng):
    op = rng.choice(("linear", "linear", "sandwich", "adamw"))
    if op == "linear":
        return dict(op=op, mode=rng.choice(("serve", "train")), rows=_log(rng, 1, 8192), k=_size(rng, 64, 4096),
                    n=_size(rng, 64, 8192), dtype=rng.choice(("bf16", "f16")),
                    act=rng.choice(("none", "silu", "gelu", "gelu_tanh", "relu")), bias=rng.random() < 0.7,
                    residual=rng.random() < 0.5)
    if op == "sandwich":
        width, dtype = _size(rng, 64, 8192), rng.choice(("bf16", "f16", "f32"))
        return dict(op=op, mode=rng.choice(("serve", "train")), rows=_log(rng, 1, min(65536, (1 << 25) // width)),
                    width=width, dtype=dtype, gate=rng.random() < 0.7, scale=rng.random() < 0.5)
    return dict(op=op, width=_size(rng, 32, 1024), hidden=_size(rng, 64, 4096), layers=_log(rng, 1, 32),
                dtype=rng.choice(("bf16", "f16", "f32")), bits=rng.choice((8, 32)))


# -------------------------------------------------------------------- inputs
def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dtype)


def _tensors(case):
    """Shapes of the stack's matrices and vectors: a gate, an up and a down projection, biases and norm weights."""
    w, h = case["width"], case["hidden"]
    return [(w, w), (h, w), (w, h)] * case["layers"], [(w,), (h,), (w,), (w,), (w,)] * case["layers"]


def _offsets(shapes):
    """Where each tensor starts in a flat buffer: at multiples of BLOCK elements."""
    at = [0]
    for s in shapes:
        at.append(at[-1] + (math.prod(s) + BLOCK - 1) // BLOCK * BLOCK)
    return at


def _views(flat, shapes):
    return [flat[a:a + math.prod(s)].view(s) for a, s in zip(_offsets(shapes), shapes)]


def _prepare_adamw(case, g):
    t, s = DTYPES[case["dtype"]], dict(case=case)
    matrices, vectors = _tensors(case)
    scale = case["width"] ** -0.5
    for kind, shapes, dtype in (("matrix", matrices, t), ("vector", vectors, torch.float32)):
        n = _offsets(shapes)[-1]
        live = torch.zeros(n, dtype=torch.bool, device="cuda")
        for v in _views(live, shapes):
            v.fill_(True)
        first = _randn(g, n, scale=scale).mul_(live)
        flat = dict(p=first.to(dtype), g=_randn(g, n, scale=1e-3).mul_(live).to(dtype))
        if dtype != torch.float32:
            flat["master"] = first
        if kind == "matrix" and case["bits"] == 8:
            # moments well into a run: the second well away from zero
            flat["m"] = _randn(g, n, scale=40.0).round_().clamp_(-127, 127).mul_(live).to(torch.int8)
            flat["v"] = torch.randint(128, 256, (n,), generator=g, device="cuda").mul_(live).to(torch.uint8)
            flat["m_scale"] = torch.rand(n // BLOCK, generator=g, device="cuda").mul_(1e-3).add_(5e-4)
            flat["v_scale"] = torch.rand(n // BLOCK, generator=g, device="cuda").mul_(4e-6).add_(2e-6)
        else:
            flat["m"] = _randn(g, n, scale=3e-4).mul_(live)
            flat["v"] = torch.rand(n, generator=g, device="cuda").mul_(1.5e-6).add_(5e-7).mul_(live)
        s[kind] = flat
        at = _offsets(shapes)
        s[kind + "_views"] = {k: [v[a // BLOCK:b // BLOCK] for a, b in zip(at, at[1:])] if k.endswith("scale")
                              else _views(v, shapes) for k, v in flat.items()}
    s["steps"] = torch.randint(100, 2000, (len(matrices) + len(vectors),), generator=g, device="cuda")
    # for the plain form: the tensor that each block of a flat buffer belongs to
    for kind, shapes, first in (("matrix", matrices, 0), ("vector", vectors, len(matrices))):
        at = torch.tensor(_offsets(shapes), device="cuda") // BLOCK
        s[kind + "_of"] = torch.repeat_interleave(torch.arange(len(shapes), device="cuda") + first, at.diff())
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "adamw":
        return _prepare_adamw(case, g)
    t, s = DTYPES[case["dtype"]], dict(case=case)
    rows = case["rows"]
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        s["x"] = _randn(g, rows, k, dtype=t)
        s["weight"] = _randn(g, n, k, dtype=t, scale=k ** -0.5)
        s["bias"] = _randn(g, n, dtype=t, scale=0.5) if case["bias"] else None
        s["residual"] = _randn(g, rows, n, dtype=t) if case["residual"] else None
        if case["mode"] == "train":
            s["dy"] = _randn(g, rows, n, dtype=t)
        return s
    width = case["width"]
    s["x"] = _randn(g, rows, width, dtype=t, scale=0.7)
    s["residual"] = _randn(g, rows, width, dtype=t, scale=2.0)
    s["weight"] = (0.5 + 0.1 * _randn(g, width)).to(t)
    s["next_weight"] = (1.0 + 0.1 * _randn(g, width)).to(t)
    s["gate"] = torch.sigmoid(_randn(g, rows, width)).to(t) if case["gate"] else None
    s["scale"] = (1.0 + 0.05 * _randn(g, width)).to(t) if case["scale"] else None
    if case["mode"] == "train":
        s["dy"] = _randn(g, rows, width, dtype=t)
        s["ds"] = _randn(g, rows, width, dtype=t)
    return s


# ----------------------------------------------------------- the plain forms
def _plain_act(z, act):
    """The activation of z and its derivative."""
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return z * sig, sig * (1.0 + z * (1.0 - sig))
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5
    if act == "gelu_tanh":
        c = (2.0 / math.pi) ** 0.5
        th = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * c * (1.0 + 3 * 0.044715 * z * z)
    if act == "relu":
        live = (z > 0).float()
        return z * live, live
    return z, torch.ones_like(z)


def _plain_linear(s):
    case, t = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if case["bias"]:
        z = z + s["bias"].float()
    y, slope = _plain_act(z, case["act"])
    if case["residual"]:
        y = y + s["residual"].float()
    if case["mode"] == "serve":
        return dict(y=y.to(t))
    dz = s["dy"].float() * slope
    out = dict(y=y.to(t), dx=(dz @ w).to(t), dweight=(dz.t() @ x).to(t))
    if case["bias"]:
        out["dbias"] = dz.sum(0).to(t)
    return out


def _plain_sandwich(s):
    case, t = s["case"], s["x"].dtype
    x, r, w, w2 = (s[k].float() for k in ("x", "residual", "weight", "next_weight"))
    gate = s["gate"].float() if case["gate"] else 1.0
    scale = s["scale"].float() if case["scale"] else 1.0
    r1 = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    xh = x * r1
    stream = (r * scale + gate * (xh * w)).to(t)  # the stream is stored, and what is stored is normalised
    f = stream.float()
    r2 = 1.0 / torch.sqrt((f * f).mean(1, keepdim=True) + EPS)
    fh = f * r2
    y = (fh * w2).to(t)
    if case["mode"] == "serve":
        return dict(y=y, stream=stream)
    dy = s["dy"].float()
    a2 = dy * w2
    g = r2 * (a2 - fh * (a2 * fh).mean(1, keepdim=True)) + s["ds"].float()
    q = g * gate
    a1 = q * w
    out = dict(y=y, stream=stream, dx=(r1 * (a1 - xh * (a1 * xh).mean(1, keepdim=True))).to(t),
               dresidual=(g * scale).to(t), dweight=(q * xh).sum(0).to(t), dnext_weight=(dy * fh).sum(0).to(t))
    if case["gate"]:
        out["dgate"] = (g * (xh * w)).to(t)
    if case["scale"]:
        out["dscale"] = (g * r).sum(0).to(t)
    return out


def _plain_values(codes, scale):
    """What the codes of an 8-bit moment stand for: t |t| (signed) or t^4 times the block's largest."""
    c = codes.float().view(-1, BLOCK)
    if codes.dtype == torch.int8:
        c = c * (1.0 / 127.0)
        return c * c.abs() * scale[:, None]
    c = c * (1.0 / 255.0)
    return c * c * (c * c) * scale[:, None]


def _plain_codes(v, signed):
    """A moment in 8 bits, a scale for each block: roots of the share of the block's largest."""
    top = v.abs().amax(1)
    share = v.abs() * (1.0 / torch.where(top > 0, top, torch.ones_like(top)))[:, None]
    if signed:
        return (torch.round(torch.sqrt(share) * 127.0) * torch.sign(v)).to(torch.int8), top
    c = torch.round(torch.sqrt(torch.sqrt(share)) * 255.0)
    return torch.maximum(c, (v > 0).float()).to(torch.uint8), top  # what is not zero stays so


def _plain_adamw(s):
    out = dict(steps=s["steps"].add_(1))
    t = s["steps"].double()
    size, root = (LR / (1.0 - BETA1 ** t)).float(), (1.0 / torch.sqrt(1.0 - BETA2 ** t)).float()
    for kind in ("matrix", "vector"):
        f = s[kind]
        eight = f["m"].dtype == torch.int8
        of, g = s[kind + "_of"], f["g"].float().view(-1, BLOCK)
        m = _plain_values(f["m"], f["m_scale"]) if eight else f["m"].view(-1, BLOCK)
        v = _plain_values(f["v"], f["v_scale"]) if eight else f["v"].view(-1, BLOCK)
        m = BETA1 * m + (1.0 - BETA1) * g
        v = BETA2 * v + (1.0 - BETA2) * (g * g)
        update = m / (torch.sqrt(v) * root[of][:, None] + ADAM_EPS) * size[of][:, None]
        p = f.get("master", f["p"]).view(-1, BLOCK)
        p = p * (1.0 - LR * DECAY) - update
        f["p"].copy_(p.view(-1))
        out[kind] = f["p"]
        if "master" in f:
            out[kind + "_master"] = f["master"].copy_(p.view(-1))
        if eight:
            for k, moment in (("m", m), ("v", v)):
                codes, scale = _plain_codes(moment, k == "m")
                f[k].copy_(codes.view(-1))
                out[kind + "_" + k + "_scale"] = f[k + "_scale"].copy_(scale)
                out[kind + "_" + k] = _plain_values(f[k], f[k + "_scale"]).view(-1).bfloat16()
        else:
            out[kind + "_m"], out[kind + "_v"] = f["m"].copy_(m.view(-1)), f["v"].copy_(v.view(-1))
    return out


# ------------------------------------------------------ the framework's calls
def _own_linear(s):
    from so3lr_b200 import layers

    case = s["case"]
    act = None if case["act"] == "none" else case["act"]
    if case["mode"] == "serve":
        return dict(y=layers.linear(s["x"], s["weight"], s["bias"], s["residual"], activation=act))
    y, saved = layers.linear_train(s["x"], s["weight"], s["bias"], s["residual"], activation=act)
    dx, dweight, dbias = layers.linear_backward(s["dy"], saved)
    out = dict(y=y, dx=dx, dweight=dweight)
    if case["bias"]:
        out["dbias"] = dbias
    return out


def _own_sandwich(s):
    from so3lr_b200 import layers

    case = s["case"]
    args = s["x"], s["residual"], s["weight"], s["next_weight"], s["gate"], s["scale"]
    y, stream = layers.sandwich_norm(*args, eps=EPS)
    if case["mode"] == "serve":
        return dict(y=y, stream=stream)
    dx, dresidual, dweight, dnext, dgate, dscale = layers.sandwich_norm_backward(s["dy"], s["ds"], stream, *args,
                                                                                 eps=EPS)
    out = dict(y=y, stream=stream, dx=dx, dresidual=dresidual, dweight=dweight, dnext_weight=dnext)
    if case["gate"]:
        out["dgate"] = dgate
    if case["scale"]:
        out["dscale"] = dscale
    return out


def _own_adamw(s):
    from so3lr_b200 import optim

    a, b = s["matrix_views"], s["vector_views"]
    few, many = [None] * len(b["p"]), [None] * len(a["p"])
    optim.adamw_step(a["p"] + b["p"], a["g"] + b["g"], a["m"] + b["m"], a["v"] + b["v"], s["steps"],
                     exp_avg_scales=a.get("m_scale", many) + few, exp_avg_sq_scales=a.get("v_scale", many) + few,
                     masters=a.get("master", many) + few, lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS,
                     weight_decay=DECAY)
    out = dict(steps=s["steps"])
    for kind in ("matrix", "vector"):
        f = s[kind]
        out[kind] = f["p"]
        if "master" in f:
            out[kind + "_master"] = f["master"]
        for k in ("m", "v"):
            if k + "_scale" in f:
                out[kind + "_" + k + "_scale"] = f[k + "_scale"]
                out[kind + "_" + k] = optim.moment_values(f[k], f[k + "_scale"], torch.bfloat16)
            else:
                out[kind + "_" + k] = f[k]
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "sandwich": _own_sandwich, "adamw": _own_adamw}[op](state)
    return {"linear": _plain_linear, "sandwich": _plain_sandwich, "adamw": _plain_adamw}[op](state)


# ---------------------------------------------------------------------- work
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        once = e * (m * k + n * k + m * n * (2 if case["residual"] else 1)) + (e * n if case["bias"] else 0)
        if case["mode"] == "serve":
            return {"bytes": once, "flops": 2 * m * k * n}
        return {"bytes": once + e * (m * n + m * k + n * k) + (e * n if case["bias"] else 0), "flops": 6 * m * k * n}
    if case["op"] == "sandwich":
        n = case["rows"] * case["width"]
        vectors = (3 if case["scale"] else 2) * e * case["width"]
        gate = 1 if case["gate"] else 0
        if case["mode"] == "serve":
            return {"bytes": n * e * (4 + gate) + vectors, "flops": 12 * n}
        return {"bytes": n * e * (8 + 2 * gate) + 2 * vectors, "flops": 50 * n}
    matrices, vectors = (sum(math.prod(s) for s in shapes) for shapes in _tensors(case))
    weights = 3 * e if e == 4 else 2 * e + 8  # gradient, parameter in and out; or the master in and out
    moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 4  # in and out; 8 bits with scales, read back in 16
    return {"bytes": int(matrices * (weights + moments) + vectors * 28), "flops": 15 * (matrices + vectors)}


# --------------------------------------------------------- 64-bit definitions
def _exact_linear(s):
    case = s["case"]
    d = {k: v.double() for k, v in s.items() if torch.is_tensor(v)}
    train = case["mode"] == "train"
    leaves = [d[k].requires_grad_(train) for k in ("x", "weight", "bias") if k in d]
    z = torch.nn.functional.linear(d["x"], d["weight"], d.get("bias"))
    fun = torch.nn.functional
    y = {"none": lambda v: v, "silu": fun.silu, "gelu": fun.gelu, "relu": fun.relu,
         "gelu_tanh": lambda v: fun.gelu(v, approximate="tanh")}[case["act"]](z)
    if case["residual"]:
        y = y + d["residual"]
    if not train:
        return dict(y=y)
    return dict(zip(("dx", "dweight", "dbias"), torch.autograd.grad(y, leaves, d["dy"])), y=y.detach())


def _exact_sandwich(s):
    case = s["case"]
    d = {k: v.double() for k, v in s.items() if torch.is_tensor(v)}
    norm = lambda v, w: v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + EPS) * w  # noqa: E731
    names = [k for k in ("x", "residual", "weight", "gate", "scale") if k in d]
    for k in names + ["next_weight"]:
        d[k].requires_grad_()
    added = norm(d["x"], d["weight"])
    if case["gate"]:
        added = added * d["gate"]
    whole = (d["residual"] * d["scale"] if case["scale"] else d["residual"]) + added
    # the stream is an output of the operator in its own type, and the second norm is of that output
    stream = whole.detach().to(s["x"].dtype).double().requires_grad_()
    y = norm(stream, d["next_weight"])
    out = dict(y=y.detach(), stream=stream.detach())
    if case["mode"] == "serve":
        return out
    ds, out["dnext_weight"] = torch.autograd.grad((y * d["dy"]).sum() + (stream * d["ds"]).sum(),
                                                  (stream, d["next_weight"]))
    out.update(zip(("d" + k for k in names), torch.autograd.grad(whole, [d[k] for k in names], ds)))
    return out


def _exact_block_codes(v, signed):
    top = v.abs().max(dim=1, keepdim=True).values
    share = torch.where(top > 0, v.abs() / top, torch.zeros_like(v))
    if signed:
        return (torch.round(share.pow(0.5) * 127) / 127).pow(2) * torch.sign(v) * top, top
    codes = torch.round(share.pow(0.25) * 255)
    return (torch.where(v > 0, codes.clamp(min=1), codes) / 255).pow(4) * top, top


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(s)
    if case["op"] == "sandwich":
        return _exact_sandwich(s)
    steps = s["steps"] + 1
    out = dict(steps=steps)
    for kind in ("matrix", "vector"):
        f = s[kind]
        eight = f["m"].dtype == torch.int8
        at = steps.double()[s[kind + "_of"]][:, None]
        fold = lambda v: v.double().view(-1, BLOCK)  # noqa: E731
        m, v, g = fold(f["m"]), fold(f["v"]), fold(f["g"])
        if eight:
            m = (m / 127).abs() * (m / 127) * f["m_scale"].double()[:, None]
            v = (v / 255).pow(4) * f["v_scale"].double()[:, None]
        m = m.lerp(g, 1 - BETA1)
        v = v.lerp(g.square(), 1 - BETA2)
        hat = m / (1 - torch.pow(BETA1, at))
        step = hat / ((v / (1 - torch.pow(BETA2, at))).sqrt() + ADAM_EPS)
        p = fold(f["master"] if "master" in f else f["p"])
        p = (p - LR * DECAY * p - LR * step).view(-1)
        out[kind] = p
        if "master" in f:
            out[kind + "_master"] = p
        for k, moment in (("m", m), ("v", v)):
            if eight:
                moment, top = _exact_block_codes(moment, k == "m")
                out[kind + "_" + k + "_scale"] = top.view(-1)
            out[kind + "_" + k] = moment.reshape(-1)
    return out
