"""The dense layer, the norms on both sides of a block and AdamW together, as a model is
trained with them: a step's results against the same formulas in torch (float64), a
captured step, a run that is stopped and taken up, and the example.

A block's results go through four roundings to bfloat16 one after another (hidden layer,
output, gate, stream), each 2^-9 of a value in the mean, and the gradients through as many
again: 2-norms within 8 * 2^-8 of the float64 formulas.
"""
import copy
import pathlib
import re
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

EPS = 1e-6


@pytest.fixture(scope="module")
def layers():
    from so3lr_b200 import layers
    return layers


@pytest.fixture(scope="module")
def optim():
    from so3lr_b200 import optim
    return optim


def _rand(seed, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


class Stack(torch.nn.Module):
    def __init__(self, layers, width, hidden, blocks, **how):
        super().__init__()
        self.norm_first = layers.rms_norm
        self.first = torch.nn.Parameter(torch.ones(width, device="cuda"))
        self.blocks = torch.nn.ModuleList(layers.SandwichBlock(width, hidden, **how) for _ in range(blocks))

    def forward(self, x):
        y, s = self.norm_first(x, self.first)
        for block in self.blocks:
            y, s = block(y, s)
        return y, s


def _stack(layers, seed=0, **how):
    torch.manual_seed(seed)
    model = Stack(layers, 96, 200, 2, **how)
    with torch.no_grad():
        for name, p in model.named_parameters():  # nothing that is 0 or 1 by chance
            p.add_(torch.randn_like(p) * (0.05 if p.dim() == 1 else 0.02))
    return model


def _plain(model, x, act):
    """The stack in float64, its parameters as leaves."""
    w = {n: p.detach().double().requires_grad_() for n, p in model.named_parameters()}
    norm = lambda v, weight: v / (v.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight  # noqa: E731
    s = x.double()
    y = norm(s, w["first"])
    for i in range(len(model.blocks)):
        b = {n.split(".")[2]: v for n, v in w.items() if n.startswith(f"blocks.{i}.")}
        h = act(y @ b["w_up"].t() + b["b_up"])
        out = norm(h @ b["w_down"].t() + b["b_down"], b["norm"])
        if "w_gate" in b:
            out = out * (y @ b["w_gate"].t() + b["b_gate"])
        s = s * b["residual_scale"] + out
        y = norm(s, b["next_norm"])
    return y, s, w


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("rows", [5, 400])
def test_block_against_formulas(layers, rows, gated):
    for name, act in (("silu", torch.nn.functional.silu), ("gelu", torch.nn.functional.gelu)):
        model = _stack(layers, activation=name, gated=gated)
        x = _rand(1, rows, 96).requires_grad_()
        y, s = model(x)
        ref_y, ref_s, w = _plain(model, x.detach(), act)
        near = lambda a, b, what: torch.testing.assert_close(  # noqa: E731
            float((a.detach().double() - b.detach()).norm() / b.detach().norm()), 0.0, atol=8 * 2.0 ** -8, rtol=0, msg=lambda m: f"{what}: {m}")
        near(y, ref_y, "y")
        near(s, ref_s, "s")
        dy, ds = _rand(2, rows, 96), _rand(3, rows, 96)
        torch.autograd.backward((y, s), (dy, ds))
        grads = torch.autograd.grad((ref_y * dy.double()).sum() + (ref_s * ds.double()).sum(), list(w.values()))
        for (n, p), g in zip(model.named_parameters(), grads):
            near(p.grad, g, n)


@pytest.mark.parametrize("bits", [32, 8])
def test_training_step_captured(layers, optim, bits):
    """Forward, backward and step in one graph do what the same calls do one by one."""
    eager, graphed = _stack(layers), _stack(layers)
    adams = [optim.AdamW(m.parameters(), lr=1e-3, moment_bits=bits) for m in (eager, graphed)]
    x, target = _rand(1, 300, 96), _rand(2, 300, 96)

    def step(model, adam):
        adam.zero_grad(set_to_none=False)
        y, s = model(x)
        loss = (y + s - target).float().square().mean()
        loss.backward()
        adam.step()
        return loss.detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for m, a in zip((eager, graphed), adams):
            for _ in range(2):
                step(m, a)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(graphed, adams[1])
    for k in range(3):
        x.copy_(_rand(10 + k, 300, 96))
        want = step(eager, adams[0])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(want, captured)
        for p, q in zip(eager.parameters(), graphed.parameters()):
            assert torch.equal(p, q)
            for key, value in adams[0].state[p].items():
                assert torch.equal(value, adams[1].state[q][key]), key


def test_run_taken_up_again(layers, optim, tmp_path):
    def step(model, adam, k):
        adam.zero_grad()
        y, s = model(_rand(k, 100, 96))
        (y * s).float().mean().backward()
        adam.step()

    model = _stack(layers)
    adam = optim.AdamW(model.parameters(), moment_bits=8)
    for k in range(2):
        step(model, adam, k)
    torch.save(dict(model=model.state_dict(), adam=adam.state_dict()), tmp_path / "run.pt")
    other = _stack(layers, seed=9)
    again = optim.AdamW(other.parameters(), moment_bits=8)
    saved = torch.load(tmp_path / "run.pt")
    other.load_state_dict(saved["model"])
    again.load_state_dict(saved["adam"])
    for k in range(2, 4):
        step(model, adam, k)
        step(other, again, k)
    assert all(torch.equal(p, q) for p, q in zip(model.parameters(), other.parameters()))


def test_deep_copies_and_other_types(layers, optim):
    model = copy.deepcopy(_stack(layers))
    half = Stack(layers, 64, 64, 1, dtype=torch.float16, activation=None)
    for m, dtype, width in ((model, torch.bfloat16, 96), (half, torch.float16, 64)):
        y, s = m(_rand(1, 2, 3, width, dtype=dtype))
        assert y.shape == s.shape == (2, 3, width) and y.dtype == dtype
        (y.float().sum() + s.float().sum()).backward()
        optim.AdamW(m.parameters()).step()
        assert all(bool(torch.isfinite(p).all()) for p in m.parameters())
    with pytest.raises(ValueError, match="activation must be one of"):
        layers.SandwichBlock(8, 8, activation="tanh")


@pytest.mark.parametrize("bits", [32, 8])
def test_example(bits):
    root = pathlib.Path(__file__).resolve().parents[1]
    out = subprocess.run([sys.executable, str(root / "examples" / "feed_forward_block.py"), "--molecules", "200", "--steps",
                          "3", "--moment-bits", str(bits)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    assert re.search(r"loss [0-9.]+ -> [0-9.]+ in 3 steps", out.stdout), out.stdout
