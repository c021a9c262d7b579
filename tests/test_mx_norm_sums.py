"""Row norms where a sum in 32 bits goes wrong: long rows of equal or equal-signed values, values far from zero, squares that
fp32 does not hold.  The bounds do not grow with the row's length.

Bound of y before the type's rounding, u = 2^-24: the sums are in 64 bits, so what is rounded to fp32 is the distance from the
mean (two subtractions), the root and its argument, the division, the scale and the bias: 8 u of |y| and of the bias.  The mean itself is off by
at most (c + 2) 2^-53 of the largest |h|, below 2^-28 for c <= 2^24 and in fact near 2^-50 for the blocked sums here; 2^-45 is allowed."""
import pytest
import torch

from diffusion_model_amd import mx

U = 2.0 ** -24


def check(kind, h, w, b, eps, got, dtype):
    h, w = h.double(), w.double()
    mean = h.mean(dim=1, keepdim=True) if kind == "layer" else torch.zeros(h.shape[0], 1, dtype=torch.float64, device=h.device)
    if kind == "layer":
        mean = mean + (h - mean).mean(dim=1, keepdim=True)  # torch's own sum of a long row
    rstd = 1 / torch.sqrt((h - mean).square().mean(dim=1, keepdim=True) + eps)
    y = (h - mean) * rstd * w
    size = y.abs()
    if b is not None:
        size, y = size + b.double().abs(), y + b.double()
    tol = 8 * U * size + (2.0 ** -45 * h.abs().amax(dim=1, keepdim=True) * rstd * w.abs() if kind == "layer" else 0)
    tol = tol + 2 * 2.0 ** -149 * rstd * w.abs()  # differences of subnormal numbers have this step
    if dtype != torch.float32:
        tol = tol + torch.finfo(dtype).eps / 2 * (y.abs() + tol)
    bad = (got.double() - y).abs() / (tol + 1e-37)
    assert bool((bad <= 1).all()), float(bad.max())


def run(kind, x, w, b, eps, residual=None):
    if kind == "rms":
        return mx.rmsnorm(x, w, residual=residual, eps=eps)
    return mx.layernorm(x, w, b, residual=residual, eps=eps)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("c", [1024, 8192, 16384, 16392, 1 << 20, (1 << 20) + 3, 1 << 24])
def test_rows_of_one_value(dev, kind, dtype, c):
    w = torch.linspace(0.5, 2, c, device=dev)
    for value in (0.1, -3.3, 1000.1):
        x = torch.full((2, c), value, device=dev).to(dtype)
        check(kind, x, w, None, 1e-5, run(kind, x, w, None, 1e-5), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("c", [1000, 1280, 4096, 8192, 16384, 20001, 1 << 20])
def test_rows_far_from_zero(dev, kind, c):
    """1000 and a spread of 2^-6: a mean rounded to fp32 would be off by 2^-9 of the spread."""
    gen = torch.Generator(device=dev).manual_seed(c)
    x = 1000 + 2.0 ** -6 * torch.randn(3, c, generator=gen, device=dev)
    w, b = 1 + 0.2 * torch.randn(c, generator=gen, device=dev), torch.randn(c, generator=gen, device=dev)
    check(kind, x, w, b if kind == "layer" else None, 1e-6, run(kind, x, w, b, 1e-6), torch.float32)
    y, h = run(kind, x, w, b, 1e-6, residual=x)
    assert torch.equal(h, x + x)
    check(kind, h, w, b if kind == "layer" else None, 1e-6, y, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("c", [40, 1280, 8192, 20001])
@pytest.mark.parametrize("scale", [1e-36, 1e-30, 1e-20, 1e20, 1e30, 1e37])
def test_rows_whose_squares_fp32_does_not_hold(dev, kind, dtype, c, scale):
    gen = torch.Generator(device=dev).manual_seed(c)
    x = (scale * torch.randn(3, c, generator=gen, device=dev).clamp(-8, 8)).to(dtype)
    w = 1 + 0.2 * torch.randn(c, generator=gen, device=dev)
    for eps in (0.0, 1e-5):
        check(kind, x, w, None, eps, run(kind, x, w, None, eps), dtype)
