"""optim.AdamW over several groups: a step that is refused changes nothing."""
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def optim():
    return pytest.importorskip("so3lr_b200.optim")


def _parameter(*shape, dtype=torch.float32):
    return torch.nn.Parameter(torch.randn(*shape, device="cuda").to(dtype))


BREAK = {
    "sparse gradient": lambda w, group: setattr(w, "grad", torch.eye(70, device="cuda").to_sparse()),
    "eps": lambda w, group: group.update(eps=0.0),
    "rate": lambda w, group: group.update(lr=-1.0),
    "rate on the CPU": lambda w, group: group.update(lr=torch.zeros(1)),
    "decay": lambda w, group: group.update(weight_decay=float("nan")),
}


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("started", [False, True])
@pytest.mark.parametrize("what", list(BREAK))
def test_refused_step_changes_nothing(optim, what, started, bits):
    """The second group's call is refused: the first group is not stepped either, no counter has moved, and
    no master has been made of weights that may still be loaded."""
    from so3lr_b200 import So3lrError
    first, second = _parameter(70, 70, dtype=torch.bfloat16), _parameter(70, 70)
    adam = optim.AdamW([dict(params=[first]), dict(params=[second], lr=1e-4)], lr=1e-3, moment_bits=bits)
    for w in (first, second):
        w.grad = torch.ones_like(w)
    if started:
        adam.step()
        for w in (first, second):
            w.grad = torch.ones_like(w)
    kept, good = [w.detach().clone() for w in (first, second)], dict(adam.param_groups[1])
    state = {w: {k: v.clone() for k, v in adam.state[w].items()} for w in (first, second) if w in adam.state}
    BREAK[what](second, adam.param_groups[1])
    with pytest.raises((ValueError, So3lrError)):
        adam.step()
    for w, before in zip((first, second), kept):
        assert torch.equal(w, before)
        assert set(adam.state.get(w, {})) == set(state.get(w, {}))
        for k, v in state.get(w, {}).items():
            assert torch.equal(adam.state[w][k], v), k
    # put right, the step is the one that was to be taken
    second.grad = torch.ones_like(second)
    adam.param_groups[1].update(good)
    adam.step()
    assert [int(adam.state[w]["step"]) for w in (first, second)] == [1 + started] * 2
    # (a step of 1e-3 is below half a unit of a bfloat16 parameter, but not of its master)
    for w, before in zip((first, second), kept):
        assert bool((adam.state[w].get("master", w) != state.get(w, {}).get("master", before)).all())


def test_check_entry_point():
    """so3lr_adamw_check says what so3lr_adamw refuses, without a GPU, and accepts the rest."""
    import ctypes as C

    from so3lr_b200 import load_library
    from test_optim_abi import _Adamw, _args
    lib = load_library()
    lib.so3lr_adamw_check.argtypes = [C.POINTER(_Adamw), C.c_char_p, C.c_size_t]
    err = C.create_string_buffer(1024)
    assert lib.so3lr_adamw_check(C.byref(_args()), err, 1024) == 0
    for change, said in ((dict(t_param=None), "param is NULL"), (dict(t_grad_dtype=2), "grad_dtype must be"),
                         (dict(t_step=(1 << 40) + 65536), "step counters overlap"), (dict(lr=-1.0), "lr must be"),
                         (dict(eps=0.0), "eps must be"), (dict(count=-1), "count must be in")):
        assert lib.so3lr_adamw_check(C.byref(_args(**change)), err, 1024) == 1
        assert said in err.value.decode(), err.value
    assert lib.so3lr_adamw_check(None, err, 1024) == 1 and b"args is NULL" in err.value
