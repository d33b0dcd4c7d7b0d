"""Rules of the row-wise feed-forward kernels' source that no run can show. No GPU."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / "so3lr_b200" / "csrc"


def _code(name):
    """The file without its comments."""
    text = (CSRC / name).read_text()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


@pytest.mark.parametrize("name", ["few_rows.cu", "rows.cu", "dense.cu", "tensor_core.cuh", "layers_common.cuh"])
def test_no_read_only_loads(name):
    """These kernels start while the kernel before them may still write what they read
    (programmatic dependent launch), so nothing of theirs is read-only for their
    lifetime, which is what non-coherent loads ask for: neither asked for by name nor
    by a pointer to const that promises to have no alias."""
    code = _code(name)
    assert not re.search(r"\.nc\b|__ldg\s*\(|\bconst\b[^,;()]*\*\s*__restrict__", code)
