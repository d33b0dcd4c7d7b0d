"""The library holds the row kernels that calls reach, and no others: their names against
the rules by which a call chooses one, stated here once more. No GPU."""
import re
import shutil
import subprocess

import pytest

TYPES = {"float": 4, "__nv_bfloat16": 2, "__half": 2}
WEIGHTS = [("float", "float")] + [(t, w) for t in ("__nv_bfloat16", "__half") for w in (t, "float")]


def _hold(width, path, size, op):
    """(lanes of a warp, 0 for a block; elements a thread)"""
    if path != "scalar":
        if width <= 64 and (path == "wide" or size == 4):
            return 8, 8
        if width <= 128:
            return 16, 8
    if width <= 512:
        return 32, 8 if width <= 256 else 16
    if path == "scalar":
        return 0, 8 if width <= 8192 else 32 if op == "gate" and width > 16384 else 16
    if op in ("norm8", "gate"):
        if path == "shifted":
            return 0, 16
        return (32, 32) if width <= 1024 else (0, 32 if op == "gate" else 16)
    return 0, 8 if width <= (1024 if path == "shifted" and op == "norm" else 4096) else 16


def _expected():
    out = set()
    for t, w in WEIGHTS:
        size = TYPES[t]
        for path in ("scalar", "wide", "shifted"):
            vec, shift = 1 if path == "scalar" else 16 // size, str(path == "shifted").lower()
            widths = range(16 // size if path == "wide" else 1, 32769, 16 // size if path == "wide" else 1)
            for width in widths:
                if width <= 16384:
                    for op in ("norm", "norm8"):
                        lanes, per = _hold(width, path, size, op)
                        out.add(f"k_rms_norm<{t}, {w}, {vec}, {per // vec}, {lanes}, {str(op == 'norm8').lower()}, {shift}>")
                    if path != "wide" or not 512 < width <= 8192:  # else the ring
                        lanes, per = _hold(width, path, size, "back")
                        threads = 256 if lanes else -(-width // (32 * per)) * 32
                        most = 256 if lanes else 512 if per == 8 and threads <= 512 else 1024
                        out.add(f"k_rms_norm_backward<{t}, {w}, {vec}, {per // vec}, {lanes}, {most}, {shift}>")
                if path == "wide" or (path == "scalar") == (width > 16384):
                    lanes, per = _hold(width, path, size, "gate")
                    out.add(f"k_gate_int8<{t}, {vec}, {per // vec}, {lanes}, {shift}>")
    return out


def test_row_kernels_are_those_that_calls_reach():
    if shutil.which("nm") is None:
        pytest.skip("nm is not installed")
    from so3lr_b200.runtime import LIB_PATH
    names = subprocess.run(["nm", "-C", str(LIB_PATH)], capture_output=True, text=True, check=True).stdout
    found = set(re.findall(r"\b(k_(?:rms_norm|rms_norm_backward|gate_int8)<[^(]*>)\(", names))
    assert found, "the library's names could not be read"
    assert found - _expected() == set(), "kernels that no call reaches"
    assert _expected() - found == set(), "kernels that are missing"
