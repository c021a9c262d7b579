"""Products of blocks at both ends of the scales' range: what bf16 and fp32 results hold there."""
import math

import pytest
import torch

from diffusion_model_amd import mx


def _one_value_a_row(dev, codes, byte, m):
    """Rows whose first value is one of `codes` under the given scale byte, the rest zero."""
    c = torch.zeros(m, 128, dtype=torch.uint8, device=dev)
    c[:, 0] = codes.to(dev).repeat(-(-m // codes.numel()))[:m]
    return mx.MXTensor(c, torch.full((m, 4), byte, dtype=torch.uint8, device=dev), 128, "mxfp8")


@pytest.mark.gpu
@pytest.mark.parametrize("m", [16, 304])  # the kernel for few tiles, the tile kernel
def test_smallest_scales(dev, m):
    """Values n 2^(byte - 136), times 2^120: exact in bf16; in fp32 too from byte 3 on, rounded to multiples of 2^-133 before."""
    w = mx.quantize(torch.full((1700, 128), 2.0 ** 120, device=dev), "mxfp4")
    codes = torch.arange(16, dtype=torch.uint8)
    for byte in (0, 1, 2, 3, 4):
        x = _one_value_a_row(dev, codes, byte, m)
        want = mx.dequantize(x)[:, :1].double() * 2.0 ** 120
        assert (mx.linear(x, w).double() == want).all()
        assert ((mx.linear(x, w, out_dtype=torch.float32).double() - want).abs() <= (2.0 ** -134 * 2.0 ** 120 if byte < 3 else 0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [16, 304])
def test_largest_scales(dev, m):
    """448 2^(byte - 127), times 2^-100: bf16 results hold them all, fp32 results those of the bytes that are written here."""
    w = mx.quantize(torch.full((1700, 128), 2.0 ** -100, device=dev), "mxfp4")
    for byte in (245, 246, 247, 254):
        x = _one_value_a_row(dev, torch.tensor([0x7e], dtype=torch.uint8), byte, m)
        want = 448 * 2.0 ** (byte - 227)
        assert (mx.linear(x, w).double() == want).all()
        assert (mx.linear(x, w, out_dtype=torch.float32).double() == (want if byte <= 246 else math.inf)).all()
    largest = torch.full((m, 128), torch.finfo(torch.float32).max, device=dev)  # no block can ask for more
    assert int(mx.quantize(largest, "mxfp8").scales[:, :4].max()) == 246 and int(mx.quantize(largest, "mxfp4").scales[:, :4].max()) == 252
