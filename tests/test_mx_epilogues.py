"""Every activation with every result type in each of the product's tile kernels, strided operands there, and every form of the
product on plain rows.  Sizes with ragged edges; the reference is in 64 bits on the device."""
import math

import pytest
import torch

from diffusion_model_amd import mx
from test_mx import PAIRS, check_linear, rows_like, unpack
from test_mx_scale_offsets import _launches_tiles

RESULTS = [torch.bfloat16, torch.float32, "mxfp8", "mxfp4"]
# What bf16 and MX results take (fp32 results of an 8-bit operand: 64 x 64 in the first row, 128 x 128 in the others):
SIZES = [(301, 1702, 160),    # 64 x 64
         (1100, 3702, 160),   # 128 x 128
         (4200, 4102, 200),   # 128 x 256 with 4-bit weights, 128 x 128 with 8-bit ones
         (4000, 3702, 4100)]  # 256 x 256


def _result(out, residual=None):
    return dict(out_format=out) if isinstance(out, str) else dict(out_dtype=out, residual=residual)


@pytest.mark.gpu
@pytest.mark.parametrize("xf,wf", PAIRS, ids=["a8w4", "a4w4", "a8w8", "a4w8"])
@pytest.mark.parametrize("m,n,k", SIZES, ids=["64", "128", "128x256", "256"])
def test_every_epilogue_of_the_tile_kernels(dev, xf, wf, m, n, k):
    assert _launches_tiles(m, n, k)
    gen = torch.Generator(device=dev).manual_seed(m + n)
    x = mx.quantize(torch.randn(m, k, generator=gen, device=dev), xf)
    w = mx.quantize(torch.randn(n, k, generator=gen, device=dev) / math.sqrt(k), wf)
    b = torch.randn(n, generator=gen, device=dev)
    xv, wv = mx.dequantize(x).double(), mx.dequantize(w).double()
    y = torch.mm(xv, wv.t().contiguous()) + b.double()
    size = torch.mm(xv.abs(), wv.abs().t().contiguous()) + b.double().abs()
    for activation in (None, "quick_gelu", "geglu"):
        wide = n // 2 if activation == "geglu" else n
        for out in RESULTS:
            res = None if isinstance(out, str) else torch.randn(m, wide, generator=gen, device=dev).to(out)
            got = mx.linear(x, w, b, activation=activation, **_result(out, res))
            if isinstance(out, str):
                assert not unpack(got)[:, wide:].any() and not got.scales[:, (wide + 31) // 32:].any()
                got = mx.dequantize(got)
            check_linear(y, size, k, got, activation, out, res, (xf, wf) != ("mxfp4", "mxfp4") and out != torch.float32)


def _inside_wider_rows(t, dev):
    codes = torch.full((t.rows, t.codes.shape[1] + 48), 0x7f, dtype=torch.uint8, device=dev)
    scales = torch.full((t.rows, t.scales.shape[1] + 12), 255, dtype=torch.uint8, device=dev)
    codes, scales = codes[:, 32:32 + t.codes.shape[1]], scales[:, 4:4 + t.scales.shape[1]]
    codes.copy_(t.codes)
    scales.copy_(t.scales)
    return mx.MXTensor(codes, scales, t.k, t.fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("xf,wf", PAIRS, ids=["a8w4", "a4w4", "a8w8", "a4w8"])
@pytest.mark.parametrize("m,n,k", SIZES, ids=["64", "128", "128x256", "256"])
def test_strided_operands_of_the_tile_kernels(dev, xf, wf, m, n, k):
    x = mx.quantize(rows_like(m, m, k).to(dev), xf)
    w = mx.quantize((rows_like(n, n, k, wide=False) / math.sqrt(k)).to(dev), wf)
    for activation, out in ((None, torch.bfloat16), ("geglu", torch.float32), ("geglu", "mxfp4")):
        want = mx.linear(x, w, activation=activation, **_result(out))
        got = mx.linear(_inside_wider_rows(x, dev), _inside_wider_rows(w, dev), activation=activation, **_result(out))
        if isinstance(out, str):
            assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
        else:
            assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("xf,wf", PAIRS, ids=["a8w4", "a4w4", "a8w8", "a4w8"])
@pytest.mark.parametrize("m,n,k", [(1, 34, 45), (3, 1282, 1279), (16, 640, 2100)])
def test_every_form_of_a_product_on_plain_rows(dev, dtype, xf, wf, m, n, k):
    """Bit for bit what quantising the rows first gives, and within the product's bound of 64 bits."""
    x = rows_like(m, m, k, dtype).to(dev)
    w = mx.quantize((rows_like(n, n, k, wide=False) / math.sqrt(k)).to(dev), wf)
    b = torch.linspace(-1, 1, n, device=dev)
    q = mx.quantize(x, xf)
    xv, wv = mx.dequantize(q).double(), mx.dequantize(w).double()
    y = torch.mm(xv, wv.t().contiguous()) + b.double()
    size = torch.mm(xv.abs(), wv.abs().t().contiguous()) + b.double().abs()
    for activation in (None, "quick_gelu", "geglu"):
        wide = n // 2 if activation == "geglu" else n
        for out in RESULTS:
            res = None if isinstance(out, str) else torch.linspace(-2, 2, m * wide, device=dev).view(m, wide).to(out)
            got = mx.linear(x, w, b, x_format=xf, activation=activation, **_result(out, res))
            want = mx.linear(q, w, b, activation=activation, **_result(out, res))
            if isinstance(out, str):
                assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
                got = mx.dequantize(got)
            else:
                assert torch.equal(got, want)
            check_linear(y, size, k, got, activation, out, res, (xf, wf) != ("mxfp4", "mxfp4") and out != torch.float32)
