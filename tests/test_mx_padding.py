"""Scale bytes behind the last block of a row belong to no value: whatever they hold, no product changes."""
import pytest
import torch

from diffusion_model_amd import mx
from test_mx import PAIRS, rows_like


def _other_padding(t, byte):
    scales = t.scales.clone()
    scales[:, (t.k + 31) // 32:] = byte
    return mx.MXTensor(t.codes, scales, t.k, t.fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("xf,wf", PAIRS, ids=["a8w4", "a4w4", "a8w8", "a4w8"])
@pytest.mark.parametrize("m,n", [(3, 70), (40, 200), (301, 1700), (1100, 3700), (4200, 4100)])
@pytest.mark.parametrize("k", [1, 33, 70, 128, 140, 1100])
def test_scales_behind_the_last_block(dev, xf, wf, m, n, k):
    x, w = mx.quantize(rows_like(m, m, k).to(dev), xf), mx.quantize(rows_like(n, n, k).to(dev), wf)
    for out in (dict(out_dtype=torch.bfloat16), dict(out_dtype=torch.float32), dict(out_format="mxfp8")):
        want = mx.linear(x, w, **out)
        for a, b in ((_other_padding(x, 255), w), (x, _other_padding(w, 255)), (_other_padding(x, 254), _other_padding(w, 254))):
            got = mx.linear(a, b, **out)
            if "out_format" in out:
                assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
            else:
                assert torch.equal(got, want)
    assert torch.equal(mx.dequantize(_other_padding(x, 255)), mx.dequantize(x))
    if m <= 16:
        plain = rows_like(m, m, k).to(dev)
        assert torch.equal(mx.linear(plain, _other_padding(w, 255), x_format=xf), mx.linear(plain, w, x_format=xf))
