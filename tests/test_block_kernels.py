"""The library holds the kernels of the norms on both sides of a block that calls reach, and no
others: their names against the rules by which a call chooses one, stated here once more.
No GPU."""
import re
import shutil
import subprocess

import pytest

TYPES = {"float": 4, "__nv_bfloat16": 2, "__half": 2}
WEIGHTS = [("float", "float")] + [(t, w) for t in ("__nv_bfloat16", "__half") for w in (t, "float")]


def _hold(width, path, size, backward):
    """(lanes of a warp, 0 for a block; elements a thread, 0: none holds the row)"""
    if path != "scalar":
        if width <= 64 and (path == "wide" or size == 4):
            return 8, 8
        if width <= 128:
            return 16, 8
    if width <= 512:
        return 32, 8 if width <= 256 else 16
    if backward and width > 4096:
        return 0, 0
    return 0, 8 if width <= 8192 else 16


def _expected():
    out = set()
    for t, w in WEIGHTS:
        size = TYPES[t]
        for path in ("scalar", "wide", "shifted"):
            vec, shift = 1 if path == "scalar" else 16 // size, str(path == "shifted").lower()
            step = 16 // size if path == "wide" else 1
            for width in range(step, 16385, step):
                lanes, per = _hold(width, path, size, False)
                out.add(f"k_sandwich<{t}, {w}, {vec}, {per // vec}, {lanes}, {shift}>")
                lanes, per = _hold(width, path, size, True)
                ring = path == "wide" and (256 if size == 2 else 2048) < width <= 8192
                if per and not ring:
                    out.add(f"k_sandwich_backward<{t}, {w}, {vec}, {per // vec}, {lanes}, {shift}>")
                if not per:
                    out.add(f"k_sandwich_backward_long<{t}, {w}, {vec if path == 'wide' else 1}>")
                if ring:
                    out.add(f"k_sandwich_backward_ring<{t}, {w}, {8 if width <= 4096 else 16}>")
                if path == "wide" and (512 if size == 2 else 4096) < width <= 8192:
                    out.add(f"k_sandwich_ring<{t}, {w}, {8 if width <= 4096 else 16}>")
    return out


def test_kernels_are_those_that_calls_reach():
    if shutil.which("nm") is None:
        pytest.skip("nm is not installed")
    from so3lr_b200.runtime import LIB_PATH
    names = subprocess.run(["nm", "-C", str(LIB_PATH)], capture_output=True, text=True, check=True).stdout
    found = set(re.findall(r"\b(k_sandwich(?:_backward)?(?:_ring|_long)?<[^(]*>)\(", names))
    assert found, "the library's names could not be read"
    assert found - _expected() == set(), "kernels that no call reaches"
    assert _expected() - found == set(), "kernels that are missing"
