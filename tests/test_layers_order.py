"""What a call of the row-wise feed-forward layers reads may have been written by the
call just before it, whose kernels may still be running when its own start."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def layers():
    from so3lr_b200 import layers
    return layers


def _codes(seed, rows, width):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-127, 128, (rows, width), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)


def test_weights_of_few_rows_made_by_the_call_before(layers):
    """Read back from 8 bits into the memory of the weights before them, and put into 8 bits."""
    n, k = 512, 2048
    x = torch.randn(4, n, device="cuda").bfloat16()
    a, sa, sb = _codes(1, 3, k), torch.ones(3, device="cuda"), torch.full((n,), 0.01, device="cuda")
    sets = [_codes(10 + i, k, n) for i in range(6)]
    scale = torch.full((k,), 1e-3, device="cuda")

    def chain(codes):
        w = layers.dequantize_int8(codes, scale)  # k x n
        down = layers.dequantize_int8(codes.view(n, k), sb)
        y = layers.feed_forward(x, w, w, down)
        c, s, _ = layers.rms_norm_int8(down, torch.ones(k, device="cuda"))
        return y, layers.int8_linear(a, sa, c, s, out_dtype=torch.float32)

    apart = []
    for codes in sets:
        w, down = (codes.float() * scale[:, None]).bfloat16(), (codes.view(n, k).float() * sb[:, None]).bfloat16()
        torch.cuda.synchronize()
        y = layers.feed_forward(x, w, w, down)
        c, s, _ = layers.rms_norm_int8(down, torch.ones(k, device="cuda"))
        torch.cuda.synchronize()
        apart.append((y, layers.int8_linear(a, sa, c, s, out_dtype=torch.float32)))
    for _ in range(20):
        for (y, z), (y1, z1) in zip([chain(codes) for codes in sets], apart):
            assert torch.equal(y, y1) and torch.equal(z, z1)


def test_weight_gradient_follows_its_rows(layers):
    """The norm's weight gradient is summed from what the kernel just before it wrote, in
    scratch that the calls before used too: gradients of scaled rows are scaled."""
    for rows, width in ((700, 96), (600, 1003), (3000, 2048)):
        s, dy = (torch.randn(rows, width, device="cuda") for _ in range(2))
        w = torch.ones(width, device="cuda")
        one = layers.rms_norm_backward(dy, s, w)[1]
        torch.cuda.synchronize()
        scaled = [dy * 2.0 ** i for i in range(8)]
        got = [layers.rms_norm_backward(d, s, w)[1] for _ in range(10) for d in scaled]
        for i, dw in enumerate(got):
            assert torch.equal(dw, one * 2.0 ** (i % 8))
