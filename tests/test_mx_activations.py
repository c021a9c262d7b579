"""Activations of the products over the whole range of their argument, against 64 bits.

The operands are zero and the bias is the argument, so the product is exact and what remains is the activation.  Relative
bounds: a gate's result has to be right where it is small, too.  m = 4 takes the kernel for few tiles, m = 301 the tile kernel."""
import math

import pytest
import torch

from diffusion_model_amd import mx
from test_mx_scale_offsets import _launches_tiles

U = 2.0 ** -24
N = 4000


def arguments(dev, low, high):
    """Both signs, dense around zero and spread over the range; every one an fp32 number."""
    tiny = torch.exp2(torch.linspace(-40, 0, N // 8, device=dev))
    wide = torch.linspace(low, high, N - 2 * tiny.numel(), device=dev)
    return torch.cat([-tiny, wide, tiny])


def product_of(dev, m, bias, **kw):
    n = bias.numel()
    assert m <= 16 or _launches_tiles(m, n, 32)
    x, w = mx.quantize(torch.zeros(m, 32, device=dev), "mxfp8"), mx.quantize(torch.zeros(n, 32, device=dev), "mxfp4")
    return mx.linear(x, w, bias, **kw)


def gelu(g):
    """g Phi(g) in 64 bits.  (torch.special.ndtr adds 1 and erf, which is 0 below -8.3.)"""
    g = g.double()
    return 0.5 * g * torch.special.erfc(-g * math.sqrt(0.5))


def check(got, want, rel, least):
    bad = (got.double() - want).abs() / (rel * want.abs() + least)
    assert bool((bad <= 1).all()), (float(bad.max()), int(bad.amax(dim=0).argmax()))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4, 301])
def test_quick_gelu_in_fp32(dev, m):
    """Exponential 2 ulp, its argument's remainder u, one sum, one product, one division, the gate's product: below 16 u.  Results
    below the smallest normal number lose bits."""
    v = arguments(dev, -60.0, 60.0)
    check(product_of(dev, m, v, activation="quick_gelu", out_dtype=torch.float32), v.double() * torch.sigmoid(1.702 * v.double()), 16 * U, 2.0 ** -126)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4, 301])
def test_quick_gelu_in_bf16(dev, m):
    """The type's rounding and 2^-12 (an exponential to 2^-24 of its argument, at most 88); past exp(88) the result is 0."""
    v = arguments(dev, -60.0, 60.0)
    check(product_of(dev, m, v, activation="quick_gelu"), v.double() * torch.sigmoid(1.702 * v.double()), 2.0 ** -8 + 2.0 ** -12, 2.0 ** -119)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4, 301])
def test_gelu_gates_in_fp32(dev, m):
    """Scaled complementary error function 4 ulp and two roundings of its argument, exponential 2 ulp and one rounding of its argument's
    remainder, three products: below 24 u for a gate of either sign."""
    g = arguments(dev, -13.0, 13.0)
    got = product_of(dev, m, torch.cat([torch.ones_like(g), g]), activation="geglu", out_dtype=torch.float32)
    check(got, gelu(g), 24 * U, 2.0 ** -126)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4, 301])
def test_gelu_gates_in_bf16(dev, m):
    """The type's rounding, and an eighth of it for the gate; a Phi below the smallest normal number may vanish (13 2^-126)."""
    g = arguments(dev, -13.0, 13.0)
    got = product_of(dev, m, torch.cat([torch.ones_like(g), g]), activation="geglu")
    check(got, gelu(g), 2.0 ** -8 + 2.0 ** -11, 2.0 ** -122)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4, 301])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_gates_that_are_huge_or_not_finite(dev, m, out):
    """g Phi(g) in IEEE arithmetic: g where Phi is 1, 0 where it is 0, NaN for -inf (-inf times 0) and NaN."""
    inf = float("inf")
    g = torch.tensor([512.0, -512.0, 1e30, -1e30, 3e38, -3e38, inf, -inf, float("nan"), 0.0], device=dev).repeat(410)
    got = product_of(dev, m, torch.cat([torch.ones_like(g), g]), activation="geglu", out_dtype=out).float().cpu()
    want = torch.tensor([512.0, 0.0, 1e30, 0.0, 3e38, 0.0, inf, float("nan"), float("nan"), 0.0]).to(out).float().repeat(410).expand(m, -1)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
