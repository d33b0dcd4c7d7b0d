"""Rules of the dense layer's, sandwich norm's and AdamW's source that no run can show. No GPU."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "so3lr_b200" / "csrc"


def _code(name):
    """The file without its comments."""
    text = (CSRC / name).read_text()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


@pytest.mark.parametrize("name", ["activation.cuh", "adamw.cu", "linear.cu", "pairs.cuh", "row_team.cuh", "sandwich.cu"])
def test_no_read_only_loads(name):
    """These kernels start while the kernel before them may still write what they read, so none of their loads is
    non-coherent, neither by name nor by a promise of no alias."""
    assert not re.search(r"\.nc\b|__ldg\s*\(|\bconst\b[^,;()]*\*\s*__restrict__", _code(name))


def test_gradients_that_products_read_are_not_evicted_first():
    """Without an activation dz is dy itself, which the two products read next: the elementwise kernel may mark dy as
    first to leave L2 only in calls with an activation, where it writes a dz of its own."""
    code = _code("linear.cu")
    kernel = code[code.index("__device__ __forceinline__ Chunk<T, kVec> load_part"):code.index("k_bias_sum(")]
    assert kernel.count("__ldcs") == 1
    assert re.search(r"if \(WIDE && ONCE\)\s*\{[^}]*__ldcs", kernel)
    loads = re.findall(r"load_part<([^>]*)>\((\w+) \+", kernel)
    assert len(loads) == 4
    assert all(args == "WIDE, kOnce" for args, _ in loads), loads
    assert "constexpr bool kOnce = ACT != SO3LR_NO_ACTIVATION;" in kernel
