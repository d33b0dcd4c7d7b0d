"""Weights put into 8 bits for the row-wise feed-forward layers. No GPU."""
import pytest

torch = pytest.importorskip("torch")
from so3lr_b200.build import torch_module  # noqa: E402

if torch_module() is None:
    pytest.skip("the layers' module is not built here", allow_module_level=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
def test_channels_without_finite_values(dtype):
    """Zeros, infinities and NaN in a channel make that channel's codes 0, and its scale 0 or NaN; the others
    are what they are alone."""
    from so3lr_b200 import layers
    torch.manual_seed(0)
    w = torch.randn(7, 45).to(dtype)
    alone = layers.quantize_weight(w)
    w[1], w[2, 3], w[3, 44], w[4, 0], w[5, 1], w[5, 2] = 0, float("inf"), -float("inf"), float("nan"), float("inf"), float("nan")
    codes, scales = layers.quantize_weight(w)
    assert codes.stride(0) == 48 and codes.shape == w.shape
    assert float(scales[1]) == 0 and bool(scales[2:6].isnan().all())
    assert bool((codes[1:6] == 0).all())
    for row in (0, 6):
        assert torch.equal(codes[row], alone[0][row]) and scales[row] == alone[1][row]
    assert int(codes[0].abs().max()) == 127


def test_ties_go_to_the_even_code():
    from so3lr_b200 import layers
    w = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5]])
    codes, scales = layers.quantize_weight(w)
    assert scales.tolist() == [1.0] and codes.tolist() == [[127, 0, 2, 2, 0, -2, -2, 126]]
