"""Measured cases of the row-wise feed-forward operators (so3lr_b200.layers).

Rows are atoms (or tokens), columns their features. Four operators:

  norm   RMS norm with the residual's addition: in training (forward and
         backward) and with its output in 8 bits (a scale for each row)
  int8   matrix product of 8-bit integers, a scale for each row of the
         activations and for each output channel, int32 sums
  gate   silu(g) * u of rows [g | u], its output in 8 bits with row scales:
         what stands between the two 8-bit products of a feed-forward block
  ffn    gated feed-forward block y = (silu(x Wg^T) * (x Wu^T)) Wd^T, forward
         alone (serving) or forward and backward (training)

`run` computes the plain form in 32 bits where `own` is false and calls the
framework where it is true.
"""
import math

import torch

own = False

EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# --------------------------------------------------------------------- cases
def listed():
    return [
        # one atom's features at a wide model's width: the call is all latency
        dict(name="norm_int8_one_row", op="norm", mode="int8", rows=1, width=2048, dtype="bf16", wf32=True),
        # the 24,000-atom water box at the wider shipped model's feature width
        dict(name="norm_int8_water_box", op="norm", mode="int8", rows=24000, width=256, dtype="bf16", wf32=True),
        # training on a batch with a width that no vector load divides
        dict(name="norm_train_odd", op="norm", mode="train", rows=3001, width=1003, dtype="f32", wf32=True),
        # training, the largest batch
        dict(name="norm_train_large", op="norm", mode="train", rows=16384, width=4096, dtype="bf16", wf32=False),
        # one row against a square weight: the weight's bytes are all there is
        dict(name="int8_one_row", op="int8", rows=1, k=4096, n=4096, dtype="bf16", bias=False),
        # a small batch, ragged in every length, float32 results with a bias
        dict(name="int8_ragged", op="int8", rows=333, k=1000, n=1531, dtype="f32", bias=True),
        # a long prompt or a large box through a wide layer
        dict(name="int8_large", op="int8", rows=8192, k=4096, n=8192, dtype="bf16", bias=False),
        # one row's hidden layer
        dict(name="gate_one_row", op="gate", rows=1, hidden=5632, dtype="bf16"),
        # the hidden layer of a large batch
        dict(name="gate_large", op="gate", rows=8192, hidden=8192, dtype="bf16"),
        # serving one row: three weights are read, nothing else counts
        dict(name="ffn_one_row", op="ffn", mode="serve", rows=1, width=2048, hidden=8192, dtype="bf16"),
        # training at the shipped models' wider feature width on the water box, hidden layer four times as wide
        dict(name="ffn_train_water_box", op="ffn", mode="train", rows=24000, width=256, hidden=1024, dtype="bf16"),
        # training, the largest; its hidden width and rows are ragged against every tile
        dict(name="ffn_train_large", op="ffn", mode="train", rows=8190, width=2048, hidden=8200, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A length between lo and hi, even over its logarithm: one in four as it falls, the others as layers have them."""
    n, step = _log(rng, lo, hi), rng.choice((1, 8, 16, 64))
    return max(lo, min(hi, n // step * step))


def draw(rng):
    op = rng.choice(("norm", "norm", "int8", "int8", "gate", "ffn", "ffn", "ffn"))
    if op == "norm":
        mode = rng.choice(("int8", "train"))
        width = _size(rng, 64, 8192)
        # the 8-bit values are compared in the type of x, which float32's bound would hold to the last bit
        dtype = rng.choice(("bf16", "f16") if mode == "int8" else ("bf16", "f16", "f32"))
        rows = _log(rng, 1, min(65536, (1 << 25) // width))
        return dict(op=op, mode=mode, rows=rows, width=width, dtype=dtype, wf32=dtype == "f32" or rng.random() < 0.5)
    if op == "int8":
        k, n = _size(rng, 64, 4096), _size(rng, 64, 8192)
        return dict(op=op, rows=_log(rng, 1, 8192), k=k, n=n, dtype=rng.choice(("bf16", "f16", "f32")),
                    bias=rng.random() < 0.5)
    if op == "gate":
        hidden = _size(rng, 64, 16384)
        return dict(op=op, rows=_log(rng, 1, min(32768, (1 << 26) // hidden)), hidden=hidden,
                    dtype=rng.choice(("bf16", "f16")))
    mode = rng.choice(("serve", "train"))
    width, hidden = _size(rng, 64, 2048), _size(rng, 64, 8192)
    return dict(op=op, mode=mode, rows=_log(rng, 1, 8192), width=width, hidden=hidden,
                dtype=rng.choice(("bf16", "f16")))


# -------------------------------------------------------------------- inputs
def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dtype)


def _codes(g, rows, width):
    """8-bit rows as the framework lays them out: row starts on 16-byte boundaries."""
    whole = torch.zeros(rows, (width + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    v = torch.randn(rows, width, generator=g, device="cuda").mul_(36.0).round_().clamp_(-127, 127)
    whole[:, :width] = v.to(torch.int8)
    return whole[:, :width]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        s["x"] = _randn(g, rows, width, dtype=t, scale=0.5)
        s["residual"] = _randn(g, rows, width, dtype=t, scale=2.0)
        s["weight"] = (1.0 + 0.1 * _randn(g, width)).to(torch.float32 if case["wf32"] else t)
        if case["mode"] == "train":
            s["dy"] = _randn(g, rows, width, dtype=t)
            s["ds"] = _randn(g, rows, width, dtype=t)
    elif case["op"] == "int8":
        s["a"] = _codes(g, case["rows"], case["k"])
        s["a_scale"] = torch.rand(case["rows"], generator=g, device="cuda").mul_(0.02).add_(0.01)
        s["b"] = _codes(g, case["n"], case["k"])
        s["b_scale"] = torch.rand(case["n"], generator=g, device="cuda").mul_(5e-4).add_(5e-4)
        s["bias"] = _randn(g, case["n"]) if case["bias"] else None
    elif case["op"] == "gate":
        s["gu"] = _randn(g, case["rows"], 2 * case["hidden"], dtype=t)
    else:
        rows, width, hidden = case["rows"], case["width"], case["hidden"]
        s["x"] = _randn(g, rows, width, dtype=t)
        s["w_gate"] = _randn(g, hidden, width, dtype=t, scale=width ** -0.5)
        s["w_up"] = _randn(g, hidden, width, dtype=t, scale=width ** -0.5)
        s["w_down"] = _randn(g, width, hidden, dtype=t, scale=hidden ** -0.5)
        if case["mode"] == "train":
            s["dy"] = _randn(g, rows, width, dtype=t)
    return s


# ----------------------------------------------------------- the plain forms
def _plain_to_int8(v):
    """Rows in 8 bits: what the codes stand for, and the scales."""
    scale = v.abs().amax(1) / 127.0
    codes = torch.round(v / torch.where(scale > 0, scale, torch.ones_like(scale))[:, None]).clamp(-127, 127)
    return codes * scale[:, None], scale


def _plain_norm(s):
    case, t = s["case"], s["x"].dtype
    stream = (s["x"].float() + s["residual"].float()).to(t)  # the stream is stored, and what is stored is normalised
    f, w = stream.float(), s["weight"].float()
    rstd = 1.0 / torch.sqrt((f * f).mean(1, keepdim=True) + EPS)
    hat = f * rstd
    if case["mode"] == "int8":
        values, scale = _plain_to_int8(hat * w)
        return dict(values=values.to(t), scale=scale, stream=stream)
    dy, ds = s["dy"].float(), s["ds"].float()
    a = dy * w
    dx = rstd * (a - hat * (a * hat).mean(1, keepdim=True)) + ds
    return dict(y=(hat * w).to(t), stream=stream, dx=dx.to(t), dw=(dy * hat).sum(0).to(s["weight"].dtype))


def _plain_int8(s):
    y = s["a"].float() @ s["b"].float().t()
    y = y * s["a_scale"][:, None] * s["b_scale"][None, :]
    if s["bias"] is not None:
        y = y + s["bias"]
    return dict(y=y.to(DTYPES[s["case"]["dtype"]]))


def _plain_gate(s):
    h = s["case"]["hidden"]
    g, u = s["gu"][:, :h].float(), s["gu"][:, h:].float()
    values, scale = _plain_to_int8(g / (1.0 + torch.exp(-g)) * u)
    return dict(values=values.to(s["gu"].dtype), scale=scale)


def _plain_ffn(s):
    t = s["x"].dtype
    x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.t(), x @ wu.t()
    sig = 1.0 / (1.0 + torch.exp(-g))
    h = g * sig * u
    y = h @ wd.t()
    if s["case"]["mode"] == "serve":
        return dict(y=y.to(t))
    dy = s["dy"].float()
    dh = dy @ wd
    du = dh * (g * sig)
    dg = dh * u * (sig * (1.0 + g * (1.0 - sig)))
    return dict(y=y.to(t), dx=(dg @ wg + du @ wu).to(t), dw_gate=(dg.t() @ x).to(t), dw_up=(du.t() @ x).to(t),
                dw_down=(dy.t() @ h).to(t))


# ------------------------------------------------------ the framework's calls
def _own(s):
    from so3lr_b200 import layers

    case = s["case"]
    if case["op"] == "norm":
        if case["mode"] == "int8":
            codes, scale, stream = layers.rms_norm_int8(s["x"], s["weight"], s["residual"], eps=EPS)
            return dict(values=layers.dequantize_int8(codes, scale, s["x"].dtype), scale=scale, stream=stream)
        y, stream = layers.rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)
        dx, dw = layers.rms_norm_backward(s["dy"], stream, s["weight"], s["ds"], eps=EPS)
        return dict(y=y, stream=stream, dx=dx, dw=dw)
    if case["op"] == "int8":
        return dict(y=layers.int8_linear(s["a"], s["a_scale"], s["b"], s["b_scale"], bias=s["bias"],
                                         out_dtype=DTYPES[case["dtype"]]))
    if case["op"] == "gate":
        codes, scale = layers.gate_int8(s["gu"])
        return dict(values=layers.dequantize_int8(codes, scale, s["gu"].dtype), scale=scale)
    if case["mode"] == "serve":
        return dict(y=layers.feed_forward(s["x"], s["w_gate"], s["w_up"], s["w_down"]))
    y, saved = layers.feed_forward_train(s["x"], s["w_gate"], s["w_up"], s["w_down"])
    dx, dwg, dwu, dwd = layers.feed_forward_backward(s["dy"], saved)
    return dict(y=y, dx=dx, dw_gate=dwg, dw_up=dwu, dw_down=dwd)


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "int8": _plain_int8, "gate": _plain_gate, "ffn": _plain_ffn}[state["case"]["op"]](state)


# ---------------------------------------------------------------------- work
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        n, we = case["rows"] * case["width"], 4 if case["wf32"] else e
        if case["mode"] == "int8":  # x, residual in; stream, values out (the codes, and what they stand for)
            return {"bytes": n * (3 * e + 1 + e) + 4 * case["rows"] + we * case["width"], "flops": 8 * n}
        return {"bytes": 7 * n * e + 2 * we * case["width"], "flops": 18 * n}
    if case["op"] == "int8":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": m * k + n * k + 4 * (m + n) + m * n * e + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if case["op"] == "gate":
        n = case["rows"] * case["hidden"]
        return {"bytes": 2 * n * e + n + n * e + 4 * case["rows"], "flops": 12 * n}
    t, d, h = case["rows"], case["width"], case["hidden"]
    if case["mode"] == "serve":
        return {"bytes": e * (2 * t * d + 3 * d * h), "flops": 6 * t * d * h}
    return {"bytes": e * (4 * t * d + 6 * d * h), "flops": 18 * t * d * h}


# --------------------------------------------------------- 64-bit definitions
def _exact_rows(v):
    top = v.abs().max(dim=1).values
    scale = top / 127
    codes = torch.where(top[:, None] > 0, torch.round(v / scale[:, None]), torch.zeros_like(v))
    return codes * scale[:, None], scale


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() for k, v in s.items() if torch.is_tensor(v)}
    if case["op"] == "norm":
        # the stream is an output of the operator in its own type, and the norm is of that output
        stream = (d["x"] + d["residual"]).to(s["x"].dtype).double().requires_grad_()
        weight = d["weight"].requires_grad_()
        y = stream * torch.rsqrt(stream.pow(2).mean(-1, keepdim=True) + EPS) * weight
        if case["mode"] == "int8":
            values, scale = _exact_rows(y.detach())
            return dict(values=values, scale=scale, stream=stream.detach())
        dx, dw = torch.autograd.grad((y * d["dy"]).sum() + (stream * d["ds"]).sum(), (stream, weight))
        return dict(y=y.detach(), stream=stream.detach(), dx=dx, dw=dw)
    if case["op"] == "int8":
        y = torch.einsum("tk,nk->tn", d["a"], d["b"]) * torch.outer(d["a_scale"], d["b_scale"])
        return dict(y=y + d["bias"] if case["bias"] else y)
    if case["op"] == "gate":
        g, u = d["gu"].chunk(2, dim=1)
        values, scale = _exact_rows(torch.nn.functional.silu(g) * u)
        return dict(values=values, scale=scale)
    leaves = [d[k].requires_grad_(case["mode"] == "train") for k in ("x", "w_gate", "w_up", "w_down")]
    x, wg, wu, wd = leaves
    y = torch.nn.functional.linear(
        torch.nn.functional.silu(torch.nn.functional.linear(x, wg)) * torch.nn.functional.linear(x, wu), wd)
    if case["mode"] == "serve":
        return dict(y=y)
    dx, dwg, dwu, dwd = torch.autograd.grad(y, leaves, d["dy"])
    return dict(y=y.detach(), dx=dx, dw_gate=dwg, dw_up=dwu, dw_down=dwd)
