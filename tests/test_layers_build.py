"""When the Python module of the row-wise feed-forward layers is compiled. No GPU, no compiler."""
import importlib.util
import types

import pytest

from so3lr_b200 import build


@pytest.fixture
def torch_of(monkeypatch, tmp_path):
    """Pretends that torch is installed in tmp_path, with or without its CUDA library."""
    def install(cuda=True, version="__version__ = '1.0'"):
        root = tmp_path / "torch"
        (root / "lib").mkdir(parents=True, exist_ok=True)
        (root / "__init__.py").write_text("")
        (root / "version.py").write_text(version)
        library = root / "lib" / "libtorch_cuda.so"
        library.write_bytes(b"") if cuda else library.unlink(missing_ok=True)
        found = importlib.util.find_spec
        monkeypatch.setattr(build.importlib.util, "find_spec", lambda name, *a: types.SimpleNamespace(
            origin=str(root / "__init__.py")) if name == "torch" else found(name, *a))
    return install


def _no_compiler(monkeypatch):
    def run(*a, **k):
        raise AssertionError("the compiler was called")
    monkeypatch.setattr(build.subprocess, "run", run)


def test_a_torch_for_cpus_only_builds_the_library_alone(monkeypatch, torch_of):
    torch_of(cuda=False)
    _no_compiler(monkeypatch)
    assert build.torch_module() is None
    assert build.build_torch_module(force=True) is None


def test_no_torch_and_no_python_headers(monkeypatch, torch_of, tmp_path):
    _no_compiler(monkeypatch)
    torch_of()
    assert build.torch_module() is not None
    with monkeypatch.context() as m:
        m.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path / "none")})
        assert build.build_torch_module(force=True) is None
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name, *a: None)
    assert build.build_torch_module(force=True) is None


def test_the_module_is_built_again_for_another_torch(monkeypatch, torch_of, tmp_path):
    """The same sources, older than the module, and a torch of another version."""
    pytest.importorskip("torch.utils.cpp_extension")
    calls = []

    def run(cmd, **k):
        calls.append(cmd)
        out.write_bytes(b"module")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "BUILD", tmp_path / "_build")
    out = tmp_path / "_layers.so"
    monkeypatch.setattr(build, "torch_module", lambda: out)
    torch_of(version="__version__ = '2.0'")
    for _ in range(3):
        assert build.build_torch_module() == out
    assert len(calls) == 1
    torch_of(version="__version__ = '2.1'")
    for _ in range(3):
        build.build_torch_module()
    assert len(calls) == 2
    out.unlink()
    build.build_torch_module()
    assert len(calls) == 3
