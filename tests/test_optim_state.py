"""optim.AdamW's load_state_dict with torch's hooks and types. No GPU."""
import copy

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def optim():
    return pytest.importorskip("so3lr_b200.optim")


def _run(optim, seed):
    """An optimiser well into a run, its state written by hand: an 8-bit matrix with a master and a float32 vector."""
    g = torch.Generator().manual_seed(seed)
    params = [torch.nn.Parameter(torch.randn(70, 70, generator=g).bfloat16()),
              torch.nn.Parameter(torch.randn(70, generator=g))]
    adam = optim.AdamW(params, moment_bits=8)
    for p in params:
        state = adam._start(p, adam.param_groups[0])
        for k, v in state.items():
            v.copy_(torch.randint(0, 100, v.shape, generator=g) + (0.123456789 if v.is_floating_point() else 0))
    return adam, params


def _same(a, b):
    assert set(a) == set(b)
    for k, v in a.items():
        assert v.dtype == b[k].dtype and torch.equal(v, b[k]), k


def test_types_and_copies(optim):
    (adam, params), (other, others) = _run(optim, 1), _run(optim, 2)
    saved = adam.state_dict()
    other.load_state_dict(saved)
    for p, q in zip(params, others):
        _same(adam.state[p], other.state[q])
        for k, v in adam.state[p].items():
            assert v.data_ptr() != other.state[q][k].data_ptr(), k
    assert {v.dtype for v in other.state[others[0]].values()} == {torch.int64, torch.int8, torch.uint8, torch.float32}


def test_hooks(optim):
    """A hook before the load may give another dictionary, one after it sees the state as loaded and may change it."""
    (adam, params), (third, thirds), (other, others) = _run(optim, 1), _run(optim, 3), _run(optim, 2)
    seen = []

    def after(optimizer):
        seen.append({k: v.dtype for k, v in optimizer.state[others[0]].items()})
        optimizer.state[others[1]]["step"].fill_(7)

    before = other.register_load_state_dict_pre_hook(lambda optimizer, state: third.state_dict())
    other.register_load_state_dict_post_hook(after)
    other.load_state_dict(adam.state_dict())
    _same(third.state[thirds[0]], other.state[others[0]])
    assert seen == [{k: v.dtype for k, v in third.state[thirds[0]].items()}]
    assert int(other.state[others[1]]["step"]) == 7 and int(third.state[thirds[1]]["step"]) != 7
    before.remove()
    other.load_state_dict(copy.deepcopy(adam.state_dict()))
    _same(adam.state[params[0]], other.state[others[0]])
    assert len(seen) == 2


def test_refused_load_leaves_no_hook(optim):
    (adam, params), (other, others) = _run(optim, 1), _run(optim, 2)
    broken = adam.state_dict()
    broken["param_groups"] = broken["param_groups"] * 2
    with pytest.raises(ValueError):
        other.load_state_dict(broken)
    other.load_state_dict(adam.state_dict())
    _same(adam.state[params[0]], other.state[others[0]])
    assert not other._optimizer_load_state_dict_pre_hooks and not other._optimizer_load_state_dict_post_hooks
