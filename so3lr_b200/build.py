"""Build libso3lr_b200.so in-tree with nvcc for sm_100a.

    python -m so3lr_b200.build [--force]

Every translation unit is compiled with
``-gencode arch=compute_100a,code=sm_100a -O3 -lineinfo`` and linked into
``so3lr_b200/libso3lr_b200.so``. nvcc cross-compiles without a GPU. The
translation units whose code depends on the model width are compiled once per
supported width (``-DSO3LR_FEATURES=128`` and ``=256``; the mixed-precision
filter kernels exist for F = 128 only). Object files are cached under
``so3lr_b200/_build`` and rebuilt when a source or header is newer. Where a torch with
CUDA is installed, the Python module of the row-wise feed-forward layers is compiled
against it and linked to the library.
"""
from __future__ import annotations

import concurrent.futures
import importlib.util
import os
import pathlib
import shutil
import subprocess
import sys
import sysconfig

HERE = pathlib.Path(__file__).resolve().parent
CSRC = HERE / "csrc"
BUILD = HERE / "_build"
LIB = HERE / "libso3lr_b200.so"
INCLUDE = HERE.parent / "include"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-O3", "-std=c++17", "-Xcompiler", "-fPIC", "-lineinfo", "-I", str(INCLUDE), "-I", str(CSRC)]
CU_FLAGS = ARCH + COMMON + ["--expt-relaxed-constexpr", "-Xptxas", "-warn-spills"]


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(path):
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libso3lr_b200")
    return path


# width-dependent translation units and the widths each is compiled for
SHAPED = {"attention.cu": (128, 256), "filter.cu": (128, 256), "node.cu": (128, 256),
          "evaluator.cu": (128, 256), "local_frame.cu": (128, 256),
          "filter_mixed.cu": (128,), "filter_tc.cu": (128,)}


def sources():
    """(source, model width or None) for every object of the library"""
    out = []
    for src in sorted(list(CSRC.glob("*.cu")) + list(CSRC.glob("*.cpp"))):
        for width in SHAPED.get(src.name, (None,)):
            out.append((src, width))
    return out


def headers():
    return sorted(list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.hpp")) + list(INCLUDE.glob("*.h")))


def _compile(unit, newest_header: float, force: bool, verbose: bool) -> pathlib.Path:
    src, width = unit
    obj = BUILD / (src.name + (f".f{width}" if width else "") + ".o")
    if not force and obj.exists() and obj.stat().st_mtime >= max(src.stat().st_mtime, newest_header):
        return obj
    cmd = [nvcc(), "-c", str(src), "-o", str(obj)] + CU_FLAGS
    if src.suffix == ".cpp":
        cmd = [nvcc(), "-x", "cu", "-c", str(src), "-o", str(obj)] + CU_FLAGS
    if width:
        cmd += [f"-DSO3LR_FEATURES={width}"]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src.name} (width {width}):\n{res.stdout}\n{res.stderr}")
    if verbose and res.stderr:
        sys.stderr.write(res.stderr)
    return obj


def torch_root() -> pathlib.Path | None:
    """The folder of the torch that `import torch` would take, without importing it."""
    spec = importlib.util.find_spec("torch")
    return pathlib.Path(spec.origin).parent if spec is not None and spec.origin else None


def torch_module() -> pathlib.Path | None:
    """The Python module of the feed-forward layers (binding/layers_binding.cpp),
    compiled against the torch that is installed. None where it cannot be: without
    torch, with one for CPUs only, or without Python's headers (the rest of the package
    needs none of them)."""
    root = torch_root()
    if root is None or not (root / "lib" / "libtorch_cuda.so").exists():
        return None
    if not (pathlib.Path(sysconfig.get_paths()["include"]) / "Python.h").exists():
        return None
    return HERE / ("_layers" + sysconfig.get_config_var("EXT_SUFFIX"))


def build_torch_module(force: bool = False) -> pathlib.Path | None:
    out = torch_module()
    if out is None:
        return None
    src, header = HERE / "binding" / "layers_binding.cpp", INCLUDE / "so3lr_b200.h"
    newest = max(f.stat().st_mtime for f in (src, header, pathlib.Path(__file__)))
    # what the module was compiled against: its binary interface is that of one torch build
    stamp, version = BUILD / "layers_module.txt", (torch_root() / "version.py").read_text()
    current = stamp.exists() and stamp.read_text() == version
    if not force and current and out.exists() and out.stat().st_mtime >= newest:
        return out
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    includes = include_paths("cuda") + [sysconfig.get_paths()["include"], str(INCLUDE)]
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", str(src), "-o", str(out),
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}"]
    cmd += [f"-I{p}" for p in includes] + [f"-L{p}" for p in library_paths("cuda")]
    cmd += [f"-L{HERE}", "-Wl,-rpath,$ORIGIN", "-lso3lr_b200", "-ltorch_python", "-ltorch", "-ltorch_cpu",
            "-ltorch_cuda", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed for {src.name}:\n{res.stdout}\n{res.stderr}")
    BUILD.mkdir(exist_ok=True)
    stamp.write_text(version)
    return out


def build(force: bool = False, verbose: bool = False) -> pathlib.Path:
    BUILD.mkdir(exist_ok=True)
    newest_header = max([h.stat().st_mtime for h in headers()] + [pathlib.Path(__file__).stat().st_mtime])
    srcs = sources()
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as pool:
        objs = list(pool.map(lambda s: _compile(s, newest_header, force, verbose), srcs))
    if force or not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        cmd = [nvcc(), "-shared", "-o", str(LIB)] + ARCH + [str(o) for o in objs] + ["-lcudart", "-ldl", "-Xlinker", "-rpath=/usr/local/cuda/lib64"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    build_torch_module(force)
    return LIB


if __name__ == "__main__":
    lib = build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(lib)
