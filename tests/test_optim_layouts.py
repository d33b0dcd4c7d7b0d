"""optim.AdamW on parameters of any layout and on several devices, as torch's own optimisers take them."""
import copy

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def optim():
    return pytest.importorskip("so3lr_b200.optim")


def _draw(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


LAYOUTS = {
    "channels last": lambda t: t.contiguous(memory_format=torch.channels_last),
    "transposed": lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
    "sliced": lambda t: torch.stack([t, t], -1)[..., 0],
    "within rows": lambda t: torch.nn.functional.pad(t, (0, 5))[..., :t.shape[-1]],
}


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_layouts(optim, layout, dtype, bits):
    """Bit for bit what the same weights do contiguously, with gradients of either layout; what lies between
    a parameter's elements is left as it was, and the saved state fits parameters of both layouts."""
    start = _draw(1, 33, 16, 3, 5).to(dtype)
    plain = torch.nn.Parameter(start.clone())
    other = torch.nn.Parameter(LAYOUTS[layout](start))
    assert not other.is_contiguous() and torch.equal(plain, other)
    storage = torch.as_strided(other.detach(), (other.untyped_storage().nbytes() // other.element_size(),), (1,), 0)
    between = storage.clone()
    between.as_strided(other.shape, other.stride(), other.storage_offset()).fill_(0)
    adams = [optim.AdamW([w], lr=1e-2, weight_decay=0.1, moment_bits=bits) for w in (plain, other)]
    for k in range(4):
        g = _draw(2 + k, *start.shape).to(dtype)
        plain.grad, other.grad = g, g.clone() if k % 2 else LAYOUTS[layout](g)
        for a in adams:
            a.step()
        if k == 1:  # each goes on with the other's state
            states = [copy.deepcopy(a.state_dict()) for a in adams]
            for a, s in zip(adams, reversed(states)):
                a.load_state_dict(s)
    assert torch.equal(plain, other) and not torch.equal(plain, start)
    for key, value in adams[0].state[plain].items():
        assert torch.equal(value, adams[1].state[other][key]), key
    storage.as_strided(other.shape, other.stride(), other.storage_offset()).fill_(0)
    assert torch.equal(storage, between)


@pytest.mark.gpu
def test_layouts_mark_and_refuse(optim):
    """A backward pass that kept the parameter from before is refused; so is a parameter whose elements share memory."""
    w = torch.nn.Parameter(_draw(1, 30, 20).t())
    loss = (w * w).sum()
    w.grad = torch.ones_like(w)
    optim.AdamW([w]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    for shared in (torch.ones(1, 8, device="cuda").expand(4, 8), torch.ones(16, device="cuda").as_strided((4, 4), (2, 1))):
        w = torch.nn.Parameter(shared)
        w.grad = torch.ones(w.shape, device="cuda")
        adam = optim.AdamW([w])
        with pytest.raises(ValueError, match="share memory"):
            adam.step()
        assert w not in adam.state and bool((w == 1).all())


@pytest.mark.gpu
def test_captured_in_another_layout(optim):
    w = torch.nn.Parameter(_draw(1, 70, 130).t())
    twin = torch.nn.Parameter(w.detach().contiguous())
    adams = [optim.AdamW([p], lr=1e-2) for p in (w, twin)]
    grads = [_draw(2 + k, 130, 70) for k in range(4)]
    w.grad, twin.grad = grads[0].clone(), grads[0].clone()
    for a in adams:
        a.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        adams[0].step()
    for g in grads[1:]:
        w.grad.copy_(g)
        graph.replay()
        twin.grad = g
        adams[1].step()
    assert torch.equal(w, twin)


class _Calls:
    """Stands in for the compiled module: records what a step asks for."""

    def __init__(self, module):
        self.uniform = module.uniform

    def adamw_steps(self, calls):
        self.calls = calls


def test_a_call_for_each_device(optim, monkeypatch):
    """A group over two devices is a call for each, in one step. No GPU: the devices are the CPU and torch's
    meta device."""
    record = _Calls(optim._layers)
    monkeypatch.setattr(optim, "_layers", record)
    params = [torch.nn.Parameter(torch.ones(n, device=d)) for n, d in ((3, "cpu"), (4, "meta"), (5, "cpu"), (6, "meta"))]
    for p in params:
        p.grad = torch.ones_like(p)
    adam = optim.AdamW([dict(params=params[:3]), dict(params=params[3:], lr=0.5)])
    adam.step()
    assert [[p.numel() for p in c[0]] for c in record.calls] == [[3, 5], [4], [6]]
    assert [c[8] for c in record.calls] == [1e-3, 1e-3, 0.5]
    for c in record.calls:
        lists = [x for x in c[:8] if isinstance(x, list)]
        assert len({t.device for x in lists for t in x if t is not None}) == 1
        assert all(len(x) == len(c[0]) for x in lists)


def test_share_memory(optim):
    """Against the elements' addresses, over random layouts of one storage. No GPU."""
    import random
    rng, storage = random.Random(0), torch.zeros(4000, dtype=torch.uint8)
    seen = [0, 0]

    def draw():
        dtype = rng.choice((torch.uint8, torch.int16, torch.float32))
        dims = [(rng.choice((1, 2, 3, 5, 8, 21, 40)), rng.randint(1, 5)) for _ in range(rng.randint(0, 3))]
        base = storage[:4000 // 4 * 4].view(dtype)
        return base.as_strided([n for _, n in dims], [s for s, _ in dims], rng.randint(0, 200) // dtype.itemsize)

    def addresses(t):
        at = torch.zeros((), dtype=torch.int64)
        for n, s in zip(t.shape, t.stride()):
            at = at[..., None] + torch.arange(n) * s
        first = (t.data_ptr() - storage.data_ptr() + at.reshape(-1, 1) * t.element_size())
        return set((first + torch.arange(t.element_size())).flatten().tolist())

    for _ in range(3000):
        a, b = draw(), draw()
        want = bool(addresses(a) & addresses(b))
        assert optim._share_memory(a, b) == want, (a.shape, a.stride(), a.data_ptr(), b.shape, b.stride(), b.data_ptr())
        seen[want] += 1
    assert min(seen) > 300


@pytest.mark.gpu
@pytest.mark.parametrize("groups", [1, 2])
def test_parameters_within_one_matrix(optim, groups):
    """Columns of one matrix are parameters of their own; a matrix and its transpose are refused, in one group or in two."""
    split = lambda params: params if groups == 1 else [dict(params=params[:1]), dict(params=params[1:])]  # noqa: E731
    whole = _draw(1, 40, 30)
    parts = [torch.nn.Parameter(whole[:, :11]), torch.nn.Parameter(whole[:, 11:])]
    twins = [torch.nn.Parameter(p.detach().contiguous()) for p in parts]
    adams = [optim.AdamW(split(p), lr=1e-2) for p in (parts, twins)]
    for k in range(3):
        for p, q in zip(parts, twins):
            p.grad = _draw(5 + k, *p.shape)
            q.grad = p.grad.clone()
        for a in adams:
            a.step()
    for p, q in zip(parts, twins):
        assert torch.equal(p, q)
    both = [torch.nn.Parameter(whole), torch.nn.Parameter(whole.t())]
    kept = whole.clone()
    for p in both:
        p.grad = torch.ones_like(p)
    adam = optim.AdamW(split(both))
    with pytest.raises(ValueError, match="share memory"):
        adam.step()
    assert torch.equal(whole, kept) and not any(adam.state.get(p) for p in both)
