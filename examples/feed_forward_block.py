"""A feed-forward sublayer over per-atom features, trained and then served in 8 bits.

    python examples/feed_forward_block.py [--molecules 8000] [--steps 60]

Rows are the atoms of a water box, columns 256 features (the wider shipped
model's width). The features are a random embedding of each atom's element and of
its distances to the nearest atoms; the block learns to add a smooth function of
them to the residual stream. Then the same weights run in 8 bits, and the script
prints how far the two forms are apart and what a call takes.
"""
from __future__ import annotations

import argparse
import pathlib
import sys

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))

import torch  # noqa: E402

from so3lr_b200 import layers  # noqa: E402
from so3lr_b200.systems import water_box  # noqa: E402

WIDTH, HIDDEN = 256, 1024


def atom_features(molecules: int) -> torch.Tensor:
    """[atoms, 256] bfloat16: cosines of random projections of (is oxygen, O-H distances, box position)."""
    box = water_box(molecules, seed=1)
    pos = torch.as_tensor(box.pos, dtype=torch.float32, device="cuda")
    oxygen = torch.as_tensor(box.z, device="cuda").eq(8).float()[:, None]
    mol = pos.view(-1, 3, 3)
    bonds = (mol[:, 1:] - mol[:, :1]).norm(dim=2).repeat_interleave(3, 0)
    raw = torch.cat([oxygen, bonds, pos / float(box.cell[0])], 1)
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.randn(raw.shape[1], WIDTH, generator=g, device="cuda")
    return torch.cos(raw @ w + torch.rand(WIDTH, generator=g, device="cuda") * 6.28).bfloat16()


def milliseconds(call, repeats: int = 20) -> float:
    call()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for _ in range(repeats):
        call()
    end.record()
    end.synchronize()
    return begin.elapsed_time(end) / repeats


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--molecules", type=int, default=8000)
    ap.add_argument("--steps", type=int, default=60)
    args = ap.parse_args()
    torch.manual_seed(0)
    x = atom_features(args.molecules)
    residual = x.roll(1, 0)
    block = layers.FeedForwardBlock(WIDTH, HIDDEN)
    target = residual + torch.sin(2 * x.float() + x.float().roll(1, 1)).bfloat16()
    master = [p.detach().float().requires_grad_() for p in block.parameters()]  # what the optimiser updates
    adam = torch.optim.Adam(master, lr=2e-3)

    def step() -> float:
        out, stream = block(x, residual)
        loss = (out + stream - target - x).float().square().mean()
        block.zero_grad()
        loss.backward()
        for p, m in zip(block.parameters(), master):
            m.grad = p.grad.float()
        adam.step()
        with torch.no_grad():
            for p, m in zip(block.parameters(), master):
                p.copy_(m)
        return float(loss.detach())

    first = step()
    for _ in range(args.steps):
        last = step()
    served = layers.Int8FeedForwardBlock(block)
    with torch.no_grad():
        out, stream = block(x, residual)
        out8, stream8 = served(x, residual)
        off = float((out8.float() - out.float()).norm() / out.float().norm())
        t16, t8 = milliseconds(lambda: block(x, residual)), milliseconds(lambda: served(x, residual))
    print(f"{x.shape[0]} atoms, {WIDTH} features, hidden {HIDDEN}: loss {first:.4f} -> {last:.4f} in {args.steps} steps")
    print(f"8-bit block: output within {100 * off:.2f} % (2-norm) of bfloat16, stream equal: "
          f"{torch.equal(stream, stream8)}; {t16:.3f} ms a call in bfloat16, {t8:.3f} ms in 8 bits")


if __name__ == "__main__":
    main()
