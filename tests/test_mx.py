"""Microscaled (MX) operands: quantisation, row norms with an MX output, products - each against its definition in 64 bits.

Quantisation is exact arithmetic (a power of two, then one rounding), so codes and scales must be equal.  Tolerances of the
others count roundings and are written where they are used; u is the unit 2^-24 of fp32.
"""
import ctypes as C
import math

import pytest
import torch

from diffusion_model_amd import _lib, mx

U = 2.0 ** -24
FMTS = ("mxfp8", "mxfp4")
EMAX = {"mxfp8": 8, "mxfp4": 2}
DTYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]


# ---- definition in 64 bits, on the CPU ------------------------------------------------------------------------------
def grid(fmt):
    if fmt == "mxfp4":
        return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    return torch.tensor([(i & 7) * 2.0 ** -9 if i < 8 else (8 + (i & 7)) * 2.0 ** ((i >> 3) - 10) for i in range(127)], dtype=torch.float64)


def encode(x, fmt):
    """[rows, k] -> (codes [rows, kp] one per value, scale bytes [rows, kp / 32])."""
    x = x.double().cpu()
    rows, k = x.shape
    b = torch.nn.functional.pad(x, (0, -k % 128)).view(rows, -1, 32)
    top = b.abs().amax(dim=2)
    bad = ~torch.isfinite(b).all(dim=2)
    e = torch.frexp(torch.where(bad | (top == 0), torch.ones_like(top), top))[1].long() - 1 - EMAX[fmt]
    e = torch.where(top == 0, torch.full_like(e, -127), e.clamp(min=-127))
    u = torch.ldexp(b, -e[..., None])
    u = torch.where(bad[..., None], torch.zeros_like(u), u)
    g = grid(fmt)
    mid = (g[1:] + g[:-1]) / 2
    lo, hi = torch.bucketize(u.abs(), mid), torch.bucketize(u.abs(), mid, right=True)
    code = torch.where(lo % 2 == 0, lo, hi)  # a midpoint goes to the even code
    sign = torch.signbit(u).long() * (128 if fmt == "mxfp8" else 8)
    return (code + sign).view(rows, -1), torch.where(bad, torch.full_like(e, 255), e + 127)


def unpack(t):
    """codes of an MXTensor, one per value."""
    c = t.codes.cpu().long()
    return c if t.fmt == "mxfp8" else torch.stack((c & 15, c >> 4), dim=2).flatten(1)


def decode(codes, scales, fmt, k):
    n = 128 if fmt == "mxfp8" else 8
    v = grid(fmt)[codes % n] * torch.where(codes >= n, -1.0, 1.0)
    s = torch.where(scales == 255, torch.full(scales.shape, float("nan"), dtype=torch.float64), torch.exp2(scales.double() - 127))
    return (v.view(codes.shape[0], -1, 32) * s[..., None]).flatten(1)[:, :k]


def values(t):
    return decode(unpack(t), t.scales.cpu().long(), t.fmt, t.k)


def rows_like(seed, rows, k, dtype=torch.float32, wide=True):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=gen)
    if wide:  # rows of very different sizes, a few channels far above the rest
        x *= torch.exp2(torch.randint(-12, 12, (rows, 1), generator=gen).float())
        x *= torch.where(torch.rand(k, generator=gen) < 0.05, 30.0, 1.0)
    return x.to(dtype)


def view_of(x, dev, off=0, extra=0):
    """The same rows inside a wider buffer: `off` elements in front, row stride k + extra."""
    if not off and not extra:
        return x.to(dev)
    buf = torch.full((x.shape[0], x.shape[1] + off + extra), float("nan"), dtype=x.dtype, device=dev)
    buf[:, off:off + x.shape[1]] = x.to(dev)
    return buf[:, off:off + x.shape[1]]


# ---- refusals (CPU) -------------------------------------------------------------------------------------------------
def test_tensors_on_the_cpu_are_refused():
    x = torch.zeros(4, 64)
    t = mx.MXTensor(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 64, "mxfp8")
    g = torch.ones(64)
    for call in (lambda: mx.quantize(x), lambda: mx.dequantize(t), lambda: mx.rmsnorm(x, g), lambda: mx.layernorm(x, g), lambda: mx.linear(x, t),
                 lambda: mx.linear(t, t)):
        with pytest.raises(RuntimeError, match="HIP device only"):
            call()


def test_mxtensor_checks_its_layout():
    codes, scales = torch.zeros(3, 128, dtype=torch.uint8), torch.zeros(3, 4, dtype=torch.uint8)
    assert mx.MXTensor(codes, scales, 100, "mxfp8").shape == (3, 100)
    assert mx.MXTensor(codes, torch.zeros(3, 8, dtype=torch.uint8), 256, "mxfp4").rows == 3
    with pytest.raises(ValueError, match="unknown MX format"):
        mx.MXTensor(codes, scales, 100, "mxfp6")
    for bad in ((codes, scales, 129, "mxfp8"), (codes, scales, 128, "mxfp4"), (codes[:2], scales, 128, "mxfp8"), (codes.float(), scales, 128, "mxfp8"),
                (codes[0], scales[0], 128, "mxfp8")):
        with pytest.raises(RuntimeError, match="MXTensor"):
            mx.MXTensor(*bad)
    with pytest.raises(ValueError, match="between 1"):
        mx.MXTensor(codes, scales, 0, "mxfp8")


def test_c_entry_points_refuse_bad_arguments_without_a_device():
    lib = _lib.lib()
    p, q = 1 << 20, (1 << 20) + 4  # never dereferenced: refused on the host
    F, B, M8, M4 = _lib.DM_F32, _lib.DM_BF16, _lib.DM_MXFP8, _lib.DM_MXFP4
    assert lib.dm_mx_quantize(p, 64, 0, 64, F, M8, None, 0, None, 0, None) == 0  # nothing to do
    for args, rc in (((None, 64, 4, 64, F, M8, p, 128, p, 4), 1), ((p, 63, 4, 64, F, M8, p, 128, p, 4), 1), ((p, 64, 4, 64, F, 6, p, 128, p, 4), 1),
                     ((p, 64, 4, 64, 7, M8, p, 128, p, 4), 1), ((p, 64, 4, 64, F, M8, p, 64, p, 4), 1), ((p, 64, 4, 64, F, M8, p, 128, p, 2), 1),
                     ((p, 64, -1, 64, F, M8, p, 128, p, 4), 1), ((p, 64, 4, 0, F, M8, p, 128, p, 4), 1), ((p, 64, 4, 64, F, M8, q, 128, p, 4), 3),
                     ((p, 64, 4, 64, F, M8, p, 136, p, 4), 3), ((p, 64, 4, 64, F, M4, p, 64, p + 1, 4), 3), ((p, 64, 4, 64, F, M4, p, 64, p, 5), 3)):
        assert lib.dm_mx_quantize(*args, None) == rc, args
    for args, rc in (((p, 128, p, 4, 4, 64, M8, None, 64, F), 1), ((p, 128, p, 4, 4, 64, M8, p, 63, F), 1), ((p, 64, p, 4, 4, 64, M8, p, 64, F), 1),
                     ((q, 128, p, 4, 4, 64, M8, p, 64, B), 3)):
        assert lib.dm_mx_dequantize(*args, None) == rc, args

    def norm(**kw):
        d = _lib.RowNormDesc(x=p, ldx=64, gamma=p, y=p, ldy=64, rows=4, c=64, dtype=F, kind=_lib.NORM_RMS, eps=1e-6)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.dm_row_norm(C.byref(d), None)
    assert lib.dm_row_norm(None, None) == 1 and norm(rows=0) == 0
    for kw in (dict(x=None), dict(gamma=None), dict(y=None), dict(ldx=63), dict(ldy=63), dict(kind=2), dict(dtype=2), dict(out_fmt=5), dict(r=p),
               dict(h=p), dict(r=p, ldr=63, h=p, ldh=64), dict(r=p, ldr=64, h=p, ldh=63), dict(out_fmt=8, ldy=128), dict(c=0), dict(rows=-1)):
        assert norm(**kw) == 1, kw
    assert norm(out_fmt=8, y=q, ldy=128, y_scales=p, ldys=4) == 3

    def gemm(**kw):
        d = _lib.MxGemmDesc(x=p, ldx=128, x_scales=p, ld_xs=4, w=p, ldw=64, w_scales=p, ld_ws=4, x_fmt=8, w_fmt=4, m=4, n=6, k=100, c=p, ldc=8,
                            c_type=B, epi=_lib.EPI_PLAIN)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.dm_mx_gemm(C.byref(d), None)
    assert lib.dm_mx_gemm(None, None) == 1 and gemm(m=0) == 0
    for kw in (dict(x=None), dict(w_scales=None), dict(c=None), dict(ldx=112), dict(ld_ws=3), dict(x_fmt=1), dict(n=0), dict(k=0), dict(m=-1), dict(m=(1 << 30) + 1), dict(n=(1 << 24) + 1), dict(ldc=5), dict(ldx=(1 << 24) + 16),
               dict(x_src=3), dict(x_src=_lib.X_BF16, ldx=99), dict(x_src=_lib.X_F32, m=17),
               dict(r=p, ldr=5), dict(epi=_lib.EPI_NCHW_F32), dict(epi=_lib.EPI_GEGLU, n=7), dict(c_type=3), dict(c_type=8, c_scales=None),
               dict(c_type=8, c_scales=p, ld_cs=4, ldc=128, r=p, ldr=8), dict(c_type=4, c_scales=p, ld_cs=4, ldc=48)):
        assert gemm(**kw) == 1, kw
    for kw in (dict(x=q), dict(ldw=72), dict(x_scales=p + 2), dict(c_type=8, c=q, ldc=128, c_scales=p, ld_cs=4)):
        assert gemm(**kw) == 3, kw


def test_c_entry_points_refuse_more_than_a_launch_holds():
    lib = _lib.lib()
    p = 1 << 20
    F, B, M8 = _lib.DM_F32, _lib.DM_BF16, _lib.DM_MXFP8
    assert lib.dm_mx_quantize(p, 1, 1 << 31, 1, F, M8, p, 128, p, 4, None) == 1  # 2^35 groups of eight values, four to a thread
    assert lib.dm_mx_quantize(p, 1, 1 << 41, 1, F, M8, p, 128, p, 4, None) == 1
    assert lib.dm_mx_dequantize(p, 128, p, 4, 1 << 31, 1, M8, p, 1, F, None) == 1
    norm = _lib.RowNormDesc(x=p, ldx=64, gamma=p, y=p, ldy=64, rows=1 << 41, c=64, dtype=F, kind=_lib.NORM_RMS, eps=1e-6)
    assert lib.dm_row_norm(C.byref(norm), None) == 1
    for bits, ld, c_type in ((8, 128, B), (4, 64, F)):
        gemm = _lib.MxGemmDesc(x=p, ldx=ld, x_scales=p, ld_xs=4, w=p, ldw=ld, w_scales=p, ld_ws=4, x_fmt=bits, w_fmt=bits, m=1 << 30, n=4096, k=128,
                               c=p, ldc=4096, c_type=c_type, epi=_lib.EPI_PLAIN)
        assert lib.dm_mx_gemm(C.byref(gemm), None) == 1


@pytest.mark.gpu
def test_python_entry_points_refuse_what_does_not_fit(dev):
    x, w = torch.zeros(4, 64, device=dev), mx.quantize(torch.zeros(6, 64, device=dev))
    odd = mx.quantize(torch.zeros(5, 64, device=dev))
    g = torch.ones(64, device=dev)
    refused = [lambda: mx.quantize(x[0]), lambda: mx.quantize(x.half()), lambda: mx.quantize(x.t()), lambda: mx.quantize(torch.zeros(1, 64, device=dev).expand(4, 64)),
               lambda: mx.dequantize(w, torch.float16), lambda: mx.rmsnorm(x, g[:32]), lambda: mx.rmsnorm(x, g.bfloat16()), lambda: mx.rmsnorm(x, g.cpu()),
               lambda: mx.rmsnorm(x, g, residual=x[:2]), lambda: mx.rmsnorm(x, g, residual=x.bfloat16()), lambda: mx.layernorm(x, g, g[:3]),
               lambda: mx.linear(x, x), lambda: mx.linear(x[:, :32].contiguous(), w), lambda: mx.linear(x, w, bias=g), lambda: mx.linear(x, odd, activation="geglu"),
               lambda: mx.linear(x, w, out_dtype=torch.float16), lambda: mx.linear(x, w, residual=torch.zeros(4, 6, device=dev)),
               lambda: mx.linear(x, w, residual=torch.zeros(4, 6, device=dev, dtype=torch.bfloat16), out_format="mxfp8")]
    for call in refused:
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: mx.quantize(x, "fp8"), lambda: mx.rmsnorm(x, g, out_format="mxfp6"), lambda: mx.linear(x, w, activation="relu"),
                 lambda: mx.quantize(x[:, :0])):
        with pytest.raises(ValueError):
            call()


# ---- quantise / dequantise ------------------------------------------------------------------------------------------
SHAPES = [(1, 1), (1, 32), (3, 31), (5, 33), (2, 127), (4, 128), (7, 129), (77, 768), (33, 1000), (1, 4096), (65, 2056), (300, 320)]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,k", SHAPES)
@pytest.mark.parametrize("off,extra", [(0, 0), (8, 16), (1, 2)], ids=["whole", "strided", "unaligned"])
def test_quantize_equals_the_definition(dev, fmt, dtype, rows, k, off, extra):
    x = rows_like(rows * 1000 + k, rows, k, dtype)
    t = mx.quantize(view_of(x, dev, off, extra), fmt)
    codes, scales = encode(x, fmt)
    assert torch.equal(t.scales.cpu().long(), scales)
    assert torch.equal(unpack(t), codes)
    want = decode(codes, scales, fmt, k)
    for dt in DTYPES:  # both types hold these values exactly
        assert torch.equal(mx.dequantize(t, dt).cpu().double(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_quantize_special_values(dev, fmt, dtype):
    """Zeros, both infinities, NaN, subnormals, the type's largest values, every midpoint between two codes, blocks at a
    power-of-two border; an infinity or a NaN spoils its own block and no other."""
    g = grid(fmt)
    mids = torch.cat([g, (g[1:] + g[:-1]) / 2])
    mids = torch.cat([mids, -mids])
    top = torch.finfo(dtype).max
    blocks = [torch.zeros(32), torch.full((32,), -0.0), torch.full((32,), top), torch.full((32,), -top), torch.full((32,), 2.0 ** -133),
              torch.full((32,), 1.5 * 2.0 ** -126), torch.arange(32) * 2.0 ** -130]
    for bad in (math.inf, -math.inf, math.nan):
        b = torch.ones(32)
        b[17] = bad
        blocks += [b, torch.ones(32)]
    for i in range(0, len(mids), 31):  # each with a leading value that fixes the scale at 2^0
        b = torch.zeros(32)
        b[0] = g[-1]
        b[1:1 + len(mids[i:i + 31])] = mids[i:i + 31]
        blocks.append(b)
    for e in (-3, 0, 5):
        for f in (1.0, 2 - 2.0 ** -7, 1 + 2.0 ** -7):
            b = torch.linspace(-1, 1, 32)
            b[3] = f * 2.0 ** e
            blocks.append(b)
    x = torch.stack([b.float() for b in blocks]).to(dtype)
    t = mx.quantize(x.to(dev), fmt)
    codes, scales = encode(x, fmt)
    assert torch.equal(t.scales.cpu().long(), scales)
    assert torch.equal(unpack(t), codes)
    got, want = mx.dequantize(t).cpu().double(), decode(codes, scales, fmt, 32)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.gpu
def test_dequantize_of_strided_codes_and_empty_matrices(dev):
    x = rows_like(1, 9, 200)
    t = mx.quantize(x.to(dev), "mxfp4")
    wide = torch.full((9, t.codes.shape[1] + 32), 0x77, dtype=torch.uint8, device=dev)
    wide[:, 16:16 + t.codes.shape[1]] = t.codes
    s = torch.full((9, t.scales.shape[1] + 8), 255, dtype=torch.uint8, device=dev)
    s[:, 4:4 + t.scales.shape[1]] = t.scales
    u = mx.MXTensor(wide[:, 16:16 + t.codes.shape[1]], s[:, 4:4 + t.scales.shape[1]], 200, "mxfp4")
    assert torch.equal(mx.dequantize(u), mx.dequantize(t))
    e = mx.quantize(torch.zeros(0, 40, device=dev))
    assert e.shape == (0, 40) and mx.dequantize(e).shape == (0, 40)
    assert mx.linear(e, mx.quantize(torch.zeros(3, 40, device=dev))).shape == (0, 3)
    assert mx.rmsnorm(torch.zeros(0, 40, device=dev), torch.ones(40, device=dev)).shape == (0, 40)


# ---- norms ----------------------------------------------------------------------------------------------------------
def norm_exact(kind, h, w, b, eps):
    """(y, size of the terms that fp32 rounds) in 64 bits."""
    h = h.double()
    mean = h.mean(dim=1, keepdim=True) if kind == "layer" else torch.zeros(h.shape[0], 1, dtype=torch.float64)
    rstd = 1 / torch.sqrt((h - mean).square().mean(dim=1, keepdim=True) + eps)
    y = (h - mean) * rstd * w.double()
    size = y.abs() + (h.abs().mean(dim=1, keepdim=True) * rstd * w.double().abs() if kind == "layer" else 0)
    if b is not None:
        size = size + b.double().abs()
        y = y + b.double()
    return y, size


def run_norm(kind, x, w, b, r, fmt, dev):
    eps = 1e-6 if kind == "rms" else 1e-5
    if kind == "rms":
        return mx.rmsnorm(x, w.to(dev), residual=r, eps=eps, out_format=fmt)
    return mx.layernorm(x, w.to(dev), None if b is None else b.to(dev), residual=r, eps=eps, out_format=fmt)


NORM_SHAPES = [(1, 1), (2, 8), (5, 31), (3, 320), (9, 512), (4, 520), (6, 1000), (3, 1283), (2, 2048), (3, 3001), (5, 4096), (2, 8192), (1, 9000), (3, 16384),
               (2, 16392), (2, 20001)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,c", NORM_SHAPES)
@pytest.mark.parametrize("residual", [False, True], ids=["plain", "residual"])
@pytest.mark.parametrize("off,extra", [(0, 0), (3, 2)], ids=["whole", "unaligned"])
def test_row_norm(dev, kind, dtype, rows, c, residual, off, extra):
    gen = torch.Generator().manual_seed(c + rows)
    x = rows_like(c, rows, c, dtype, wide=False) * 3 + 0.5
    r = (rows_like(c + 1, rows, c, dtype, wide=False) * 2).to(dtype) if residual else None
    w, b = 1 + 0.3 * torch.randn(c, generator=gen), (torch.randn(c, generator=gen) if kind == "layer" and c % 2 == 0 else None)
    xd = view_of(x, dev, off, extra)
    got = run_norm(kind, xd, w, b, None if r is None else view_of(r, dev, off, extra), None, dev)
    h = x
    if residual:
        got, hd = got
        h = (x.float() + r.float()).to(dtype)  # one fp32 addition, one rounding
        assert torch.equal(hd.cpu(), h)
    y, size = norm_exact(kind, h, w, b, 1e-6 if kind == "rms" else 1e-5)
    # A sum over the row: at most ceil(c / 2048) * 8 + 10 additions behind each other (a thread's own, then the threads'; twice
    # that for rows past 16384 with a loop of 256 threads is covered by the first term); the square root halves the sum's
    # error, the layer norm's mean enters as it is; three or four roundings of the result, then that of the type.
    depth = 8 * math.ceil(c / 2048) + 10
    if c <= 1024:
        depth = 8 * math.ceil(c / 512) + 10
    tol = (depth + 6) * U * size + (torch.finfo(dtype).eps / 2 * y.abs() if dtype != torch.float32 else 0)
    err = (got.cpu().double() - y).abs()
    assert bool((err <= tol + 1e-30).all()), float((err / (tol + 1e-30)).max())
    # an MX output is the quantisation of the unrounded fp32 result, code for code
    plain = run_norm(kind, h.float().to(dev), w, b, None, None, dev)
    for fmt in FMTS:
        q = run_norm(kind, xd, w, b, None if r is None else view_of(r, dev, off, extra), fmt, dev)
        q = q[0] if residual else q
        want = mx.quantize(plain, fmt)
        assert torch.equal(q.scales, want.scales) and torch.equal(q.codes, want.codes)


@pytest.mark.gpu
def test_row_norm_of_rows_that_are_not_finite_or_all_zero(dev):
    x = rows_like(3, 6, 256, wide=False)
    x[1, 7], x[2, 9], x[4] = math.inf, math.nan, 0.0
    w = torch.ones(256)
    y = mx.rmsnorm(x.to(dev), w.to(dev)).cpu()
    assert torch.isnan(y[2]).all() and torch.isnan(y[1, 7]) and (y[1, :7] == 0).all() and (y[4] == 0).all()
    good = [0, 3, 5]
    ref, size = norm_exact("rms", x[good], w, None, 1e-6)
    assert bool(((y[good].double() - ref).abs() <= 24 * U * size).all())
    q = mx.rmsnorm(x.to(dev), w.to(dev), out_format="mxfp8")
    v = mx.dequantize(q).cpu()
    assert torch.isnan(v[2]).all() and torch.isnan(v[1, :32]).all() and (v[1, 32:] == 0).all() and (v[4] == 0).all() and torch.isfinite(v[good]).all()


@pytest.mark.gpu
def test_row_norm_in_place_through_the_c_entry(dev):
    """h may be the residual itself, y may be x; rows behind the last one and columns behind the row stay as they are."""
    lib = _lib.lib()
    for c in (320, 20000):  # rows in registers, rows in a loop
        x, r = rows_like(5, 4, c, wide=False), rows_like(6, 4, c, wide=False)
        xb, rb = torch.full((6, c + 8), 7.0, device=dev), torch.full((6, c + 8), 7.0, device=dev)
        xb[:4, :c], rb[:4, :c] = x.to(dev), r.to(dev)
        g = torch.ones(c, device=dev)
        d = _lib.RowNormDesc(x=xb.data_ptr(), ldx=c + 8, r=rb.data_ptr(), ldr=c + 8, h=rb.data_ptr(), ldh=c + 8, gamma=g.data_ptr(), y=xb.data_ptr(),
                             ldy=c + 8, rows=4, c=c, dtype=_lib.DM_F32, kind=_lib.NORM_LAYER, eps=1e-5)
        _lib.check(lib.dm_row_norm(C.byref(d), torch.cuda.current_stream(dev).cuda_stream))
        want, h = mx.layernorm(x.to(dev), g, residual=r.to(dev))
        assert torch.equal(rb[:4, :c], h) and torch.equal(xb[:4, :c], want)
        for t in (xb, rb):
            assert (t[4:] == 7).all() and (t[:, c:] == 7).all()


# ---- products -------------------------------------------------------------------------------------------------------
def product(x, w, bias):
    """x w^T + bias in 64 bits and the sum of the terms' sizes."""
    x, w = values(x), values(w)
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, size


def check_linear(y, size, k, got, activation, out, residual, scaled):
    """Elementwise bound.  fp32 sums of k products in any order: (k + 2) u of the terms' sizes.  The scaled instructions add
    the products of 64 values of e4m3 operands with a window that ends about 2^-16 below the largest of them: up to 64 of
    them lose less than 2^-16 of the largest term each instruction, so 2^-13 of the terms' sizes is a bound with room.  Then
    the activation (slopes at most 1.13 and 1.1; its fp32 form within 2^-15 of its argument in bf16 and MX results, 8 u in fp32)
    and the rounding of the result's type."""
    err = size * ((k + 2) * U + (2.0 ** -13 if scaled else 0))
    if activation == "geglu":
        n = y.shape[1] // 2
        v, g, ev, eg = y[:, :n], y[:, n:], err[:, :n], err[:, n:]
        gelu = g * torch.special.ndtr(g)
        own = g.abs() * (2.0 ** -15 if out != torch.float32 else 16 * U)
        err = ev * (gelu.abs() + 1.13 * eg + own) + v.abs() * (1.13 * eg + own)
        y = v * gelu
    elif activation == "quick_gelu":
        s = y * torch.sigmoid(1.702 * y)
        err = 1.1 * err + s.abs() * (8 + 2 * y.abs()) * 4 * U
        y = s
    if residual is not None:
        y = y + residual.double()
        err = err + 2 * U * y.abs()
    got = got.double()
    err = err + 1e-37
    if isinstance(out, str):
        # the block's step at the value: half a code, an eighth / a quarter where the largest codes saturate
        b = torch.nn.functional.pad(y.abs() + err, (0, -y.shape[1] % 32)).view(y.shape[0], -1, 32)
        step = torch.exp2(torch.floor(torch.log2(b.amax(dim=2).clamp(min=1e-300))) - EMAX[out]).repeat_interleave(32, dim=1)[:, :y.shape[1]]
        rel, least = (0.125, 2.0 ** -10) if out == "mxfp8" else (0.25, 0.25)
        err = err + rel * (y.abs() + err) + least * step
    elif out == torch.bfloat16:
        err = err + torch.finfo(out).eps / 2 * (y.abs() + err)
    bad = (got - y).abs() / err
    assert bool((bad <= 1).all()), float(bad.max())


PRODUCTS = [(1, 1, 1), (1, 40, 32), (2, 17, 64), (3, 130, 100), (7, 64, 4096), (16, 96, 129), (17, 33, 300), (31, 500, 256), (64, 64, 128), (65, 66, 640),
            (77, 768, 768), (130, 258, 1000), (200, 320, 320), (256, 512, 384)]
PAIRS = [("mxfp8", "mxfp4"), ("mxfp4", "mxfp4"), ("mxfp8", "mxfp8"), ("mxfp4", "mxfp8")]


@pytest.mark.gpu
@pytest.mark.parametrize("xf,wf", PAIRS, ids=["a8w4", "a4w4", "a8w8", "a4w8"])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32, "mxfp8", "mxfp4"], ids=["bf16", "f32", "mx8", "mx4"])
def test_linear(dev, xf, wf, m, n, k, out):
    x = mx.quantize(rows_like(m + k, m, k).to(dev), xf)
    w = mx.quantize((rows_like(n + k, n, k, wide=False) / math.sqrt(k)).to(dev), wf)
    gen = torch.Generator().manual_seed(n)
    scaled = (xf, wf) != ("mxfp4", "mxfp4") and out != torch.float32
    for activation in (None, "quick_gelu", "geglu"):
        if activation == "geglu" and n % 2:
            continue
        wide = n // 2 if activation == "geglu" else n
        bias = torch.randn(n, generator=gen) if (m + n) % 2 else None
        res = torch.randn(m, wide, generator=gen).to(out) if not isinstance(out, str) and m % 2 else None
        kw = dict(out_format=out) if isinstance(out, str) else dict(out_dtype=out, residual=None if res is None else res.to(dev))
        got = mx.linear(x, w, None if bias is None else bias.to(dev), activation=activation, **kw)
        y, size = product(x, w, bias)
        if isinstance(out, str):
            assert got.shape == (m, wide)
            pad = unpack(got)[:, wide:]  # what the next product reads behind column n
            assert not pad.any() and not got.scales[:, (wide + 31) // 32:].any()
            got = mx.dequantize(got)
        check_linear(y, size, k, got.cpu(), activation, out, res, scaled)


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_linear_keeps_to_its_columns_and_rows(dev, out):
    """Strided operands, result and residual inside wider buffers (C entry): nothing outside the result is written."""
    for m, n, k in ((5, 70, 200), (66, 128, 256), (130, 131, 128)):
        x, w = mx.quantize(rows_like(1, m, k).to(dev), "mxfp8"), mx.quantize(rows_like(2, n, k).to(dev), "mxfp4")
        want = mx.linear(x, w, out_dtype=out, residual=torch.ones(m, n, dtype=out, device=dev))
        for off, extra in ((0, 16), (8, 8), (1, 3)):
            ld = n + off + extra
            buf, res = torch.full((m + 2, ld), 9.0, dtype=out, device=dev), torch.ones(m, ld, dtype=out, device=dev)
            cb = torch.full((m, x.codes.shape[1] + 16), 0x7f, dtype=torch.uint8, device=dev)
            cb[:, :x.codes.shape[1]] = x.codes
            d = _lib.MxGemmDesc(x=cb.data_ptr(), ldx=cb.shape[1], x_scales=x.scales.data_ptr(), ld_xs=x.scales.shape[1], w=w.codes.data_ptr(),
                                ldw=w.codes.shape[1], w_scales=w.scales.data_ptr(), ld_ws=w.scales.shape[1], x_fmt=8, w_fmt=4, m=m, n=n, k=k,
                                r=res[:, off:].data_ptr(), ldr=ld, c=buf[:, off:].data_ptr(), ldc=ld,
                                c_type=_lib.DM_F32 if out == torch.float32 else _lib.DM_BF16, epi=_lib.EPI_PLAIN)
            _lib.check(_lib.lib().dm_mx_gemm(C.byref(d), torch.cuda.current_stream(dev).cuda_stream))
            assert torch.equal(buf[:m, off:off + n], want)
            assert (buf[m:] == 9).all() and (buf[:, :off] == 9).all() and (buf[:, off + n:] == 9).all()


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32, "mxfp8"], ids=["bf16", "f32", "mx8"])
@pytest.mark.parametrize("m", [3, 70])
def test_linear_nan_stays_in_its_row(dev, m, out):
    x = rows_like(1, m, 300, wide=False)
    x[1, 40], x[2, 299] = math.nan, math.inf
    for xf in FMTS:
        w = mx.quantize(rows_like(2, 64, 300, wide=False).to(dev), "mxfp4")
        y = mx.linear(x.to(dev), w, x_format=xf, **(dict(out_format=out) if isinstance(out, str) else dict(out_dtype=out)))
        y = (mx.dequantize(y) if isinstance(out, str) else y).cpu()
        assert torch.isnan(y[1:3]).all() and torch.isfinite(y[:1]).all() and torch.isfinite(y[3:]).all()
        wb = rows_like(2, 64, 300, wide=False)
        wb[5, 3] = math.inf
        y = mx.linear(x[3:].to(dev) if m > 3 else x[:1].to(dev), mx.quantize(wb.to(dev), "mxfp8"), x_format=xf).cpu()
        assert torch.isnan(y[:, 5]).all() and torch.isfinite(y[:, :5]).all() and torch.isfinite(y[:, 6:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("xf,wf", PAIRS, ids=["a8w4", "a4w4", "a8w8", "a4w8"])
@pytest.mark.parametrize("m,n", [(1100, 1100), (4200, 4100)])  # the tile kernels
def test_linear_nan_stays_in_its_row_and_column_of_a_tile(dev, xf, wf, m, n):
    x, w = torch.ones(m, 200, device=dev), torch.ones(n, 200, device=dev)
    x[7, 150], w[33, 0] = math.nan, math.inf
    for out in DTYPES:
        y = mx.linear(mx.quantize(x, xf), mx.quantize(w, wf), out_dtype=out)
        bad = torch.isnan(y)
        assert bad[7].all() and bad[:, 33].all() and int(bad.sum()) == m + n - 1 and (y[~bad] == 200).all()


@pytest.mark.gpu
@pytest.mark.parametrize("xf,wf", PAIRS, ids=["a8w4", "a4w4", "a8w8", "a4w8"])
@pytest.mark.parametrize("m", [4, 1100])
def test_linear_extreme_scales(dev, xf, wf, m):
    """Blocks at both ends of the scales' range: 128 products 2^x 2^w, exact in every type."""
    for ex, ew in ((-120, 120), (-60, -60), (100, -120), (-125, 126), (126, -125), (-127 + EMAX[xf], 100)):
        x, w = torch.full((m, 128), 2.0 ** ex, device=dev), torch.full((1100, 128), 2.0 ** ew, device=dev)
        for out in DTYPES:
            y = mx.linear(mx.quantize(x, xf), mx.quantize(w, wf), out_dtype=out)
            assert (y.double() == 2.0 ** (ex + ew + 7)).all(), (ex, ew, out)


@pytest.mark.gpu
@pytest.mark.parametrize("xf,wf", PAIRS, ids=["a8w4", "a4w4", "a8w8", "a4w8"])
@pytest.mark.parametrize("m", [4, 1100])
def test_linear_smallest_codes_of_the_smallest_scale(dev, xf, wf, m):
    """Blocks of scale 2^-127 with values below fp32's and bf16's normal range next to large ones: every sum below is exact in
    fp32 (64 terms of 2 and 64 of 2^-11, or 64 of 2^-5 and 64 of 2^-8), and one rounding away in bf16."""
    small = -131 if xf == "mxfp8" else -128
    x = torch.full((m, 128), 2.0 ** (-127 + EMAX[xf]), device=dev)
    x[:, ::2] = 2.0 ** small
    xq, wq = mx.quantize(x, xf), mx.quantize(torch.full((1100, 128), 2.0 ** 120, device=dev), wf)
    assert torch.equal(mx.dequantize(xq), x)
    sums = 64 * (2.0 ** (EMAX[xf] - 7) + 2.0 ** (small + 120))
    assert (mx.linear(xq, wq, out_dtype=torch.float32).double() == sums).all()
    assert ((mx.linear(xq, wq).double() - sums).abs() <= sums * (2.0 ** -8 + 2.0 ** -13)).all()  # the scaled sums, then bf16


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4, 40, 1100])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_geglu_gates_far_from_zero(dev, m, out):
    """gelu(-512) is 0 and gelu(512) is 512: the polynomial's ends are held where they pass 0 and 1 to 2^-32."""
    x, w = torch.ones(m, 128, device=dev), torch.ones(256, 128, device=dev)
    w[128:] = 4
    w[192:] = -4
    y = mx.linear(mx.quantize(x, "mxfp4"), mx.quantize(w, "mxfp4"), activation="geglu", out_dtype=out)
    assert (y[:, :64] == 65536).all() and (y[:, 64:].abs() <= 65536 * 2.0 ** -32).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("xf", FMTS)
@pytest.mark.parametrize("m,n,k", [(1, 1280, 1280), (1, 33, 45), (4, 640, 1000), (16, 320, 8192), (40, 64, 320), (600, 128, 256)])
def test_linear_of_plain_rows_quantises_them(dev, dtype, xf, m, n, k):
    """Rows in fp32 / bf16 give bit for bit what quantising them first gives."""
    x = rows_like(m, m, k, dtype).to(dev)
    w = mx.quantize((rows_like(n, n, k, wide=False) / math.sqrt(k)).to(dev), "mxfp4")
    b = torch.linspace(-1, 1, n, device=dev)
    for kw in (dict(), dict(out_dtype=torch.float32, activation="quick_gelu"), dict(out_format="mxfp8")):
        a, c = mx.linear(x, w, b, x_format=xf, **kw), mx.linear(mx.quantize(x, xf), w, b, **kw)
        if "out_format" in kw:
            assert torch.equal(a.codes, c.codes) and torch.equal(a.scales, c.scales)
        else:
            assert torch.equal(a, c)


@pytest.mark.gpu
def test_linear_large_equals_blocks_of_it(dev):
    """Every row and column of a product that fills the chip, against products of pieces of it (exact sums: 4-bit operands with
    small scales), and against 64 bits on a sample of rows."""
    m, n, k = 1000, 2100, 1100
    x, w = rows_like(1, m, k, wide=False), rows_like(2, n, k, wide=False)
    xq, wq = mx.quantize(x.to(dev), "mxfp4"), mx.quantize(w.to(dev), "mxfp4")
    whole = mx.linear(xq, wq, out_dtype=torch.float32)
    for r in (0, 1, 255, 256, 511, 999):
        part = mx.linear(mx.quantize(x[r:r + 1].to(dev), "mxfp4"), wq, out_dtype=torch.float32)
        y, size = product(mx.quantize(x[r:r + 1].to(dev), "mxfp4"), wq, None)
        for got in (whole[r:r + 1], part):
            assert bool(((got.cpu().double() - y).abs() <= (k + 2) * U * size).all())


# ---- offsets and grids past 32 bits ---------------------------------------------------------------------------------
@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """Rows 2^24 bytes apart in buffers of 5 GB and results of 2.6 GB give what the same rows side by side give."""
    rows, k, ld = 300, 1283, 1 << 24
    x = rows_like(5, rows, k, torch.bfloat16).to(dev)
    far = torch.zeros(rows * ld // 2, dtype=torch.bfloat16, device=dev).view(rows, ld // 2)[:, 7:7 + k]
    far.copy_(x)
    g = torch.linspace(0.5, 2, k, device=dev)
    assert torch.equal(mx.rmsnorm(far, g), mx.rmsnorm(x, g))
    (a, h), (b, i) = mx.layernorm(far, g, residual=far, out_format="mxfp8"), mx.layernorm(x, g, residual=x, out_format="mxfp8")
    assert torch.equal(h, i) and torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    a, b = mx.quantize(far, "mxfp8"), mx.quantize(x, "mxfp8")
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    few = mx.quantize(x[:4], "mxfp4")
    assert torch.equal(mx.linear(far[-16:], few), mx.linear(x[-16:], few))  # plain rows
    del far
    buf = torch.zeros(rows * ld, dtype=torch.uint8, device=dev).view(rows, ld)
    buf[:, :b.codes.shape[1]], buf[:, 4096:4096 + b.scales.shape[1]] = b.codes, b.scales
    wide = mx.MXTensor(buf[:, :b.codes.shape[1]], buf[:, 4096:4096 + b.scales.shape[1]], k, "mxfp8")
    assert torch.equal(mx.dequantize(wide), mx.dequantize(b))
    w = mx.quantize(rows_like(6, 1000, k, wide=False).to(dev), "mxfp4")
    for out in DTYPES:
        assert torch.equal(mx.linear(wide, w, out_dtype=out), mx.linear(b, w, out_dtype=out))  # as the left operand: tiles
        assert torch.equal(mx.linear(w, wide, out_dtype=out), mx.linear(w, b, out_dtype=out))  # as the right one
        assert torch.equal(mx.linear(few, wide, out_dtype=out), mx.linear(few, b, out_dtype=out))  # and with few rows
    del buf, wide
    m, n, k = 65600, 20000, 96
    xq, wq = mx.quantize(rows_like(7, m, k, wide=False).to(dev), "mxfp8"), mx.quantize(rows_like(8, n, k, wide=False).to(dev), "mxfp4")
    tail = mx.MXTensor(xq.codes[-700:], xq.scales[-700:], k, "mxfp8")
    for kw in (dict(), dict(out_dtype=torch.float32)):
        assert torch.equal(mx.linear(xq, wq, **kw)[-700:], mx.linear(tail, wq, **kw))


@pytest.mark.gpu
def test_row_norm_of_more_rows_than_a_launch_holds(dev):
    """2^23 blocks of a row each per launch: the rows before, at and behind the seam, and the last ones."""
    rows, c = (1 << 23) + 1000, 1027
    x = torch.empty(rows, c, dtype=torch.bfloat16, device=dev)
    parts = [slice(0, 300), slice((1 << 23) - 300, (1 << 23) + 300), slice(rows - 300, rows)]
    for i, part in enumerate(parts):
        x[part] = rows_like(i, x[part].shape[0], c, torch.bfloat16).to(dev)
    g, b = torch.linspace(0.5, 2, c, device=dev), torch.linspace(-1, 1, c, device=dev)
    y = mx.layernorm(x, g, b)
    for part in parts:
        assert torch.equal(y[part], mx.layernorm(x[part], g, b))


# ---- together, streams, graphs --------------------------------------------------------------------------------------
def feed_forward(x, h, g, w1, b1, w2, b2):
    """norm -> gated product -> product + residual, as a quantised transformer block runs them."""
    a, h = mx.rmsnorm(x, g, residual=h, out_format="mxfp8")
    u = mx.linear(a, w1, b1, activation="geglu", out_format="mxfp8")
    return mx.linear(u, w2, b2, residual=h)


def ff_inputs(dev, rows, c):
    x, h = rows_like(1, rows, c, torch.bfloat16, wide=False).to(dev), rows_like(2, rows, c, torch.bfloat16, wide=False).to(dev)
    w1 = mx.quantize((rows_like(3, 8 * c, c, wide=False) / math.sqrt(c)).to(dev), "mxfp4")
    w2 = mx.quantize((rows_like(4, c, 4 * c, wide=False) / math.sqrt(4 * c)).to(dev), "mxfp4")
    return x, h, torch.linspace(0.5, 1.5, c, device=dev), w1, torch.linspace(-1, 1, 8 * c, device=dev), w2, torch.linspace(1, -1, c, device=dev)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 77, 300])
def test_feed_forward_against_64_bits(dev, rows):
    args = ff_inputs(dev, rows, 320)
    got = feed_forward(*args).cpu().double()
    x, h, g, w1, b1, w2, b2 = [values(a) if isinstance(a, mx.MXTensor) else a.cpu().double() for a in args]
    h = (x.float() + h.float()).bfloat16().double()
    a = h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-6) * g
    a = decode(*encode(a, "mxfp8"), "mxfp8", 320)
    v, gate = (a @ w1.t() + b1).chunk(2, dim=1)
    u = v * gate * torch.special.ndtr(gate)
    u = decode(*encode(u, "mxfp8"), "mxfp8", 1280)
    y = u @ w2.t() + b2 + h
    # Roundings that fall on the other side of a border (the norm's and the product's fp32 errors against 64 bits) move a
    # value by at most an eighth of itself; with at most one such value in 2^8 the sum of 1280 moves by less than 2^-8 of its
    # terms' sizes; then the bf16 rounding of the result.
    size = u.abs() @ w2.abs().t()
    assert bool(((got - y).abs() <= 2.0 ** -8 * size + 2.0 ** -8 * y.abs()).all())


@pytest.mark.gpu
def test_feed_forward_on_another_stream_and_in_a_graph(dev):
    args = ff_inputs(dev, 40, 320)
    want = feed_forward(*args)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = feed_forward(*args)
    torch.cuda.current_stream(dev).wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    x = args[0].clone()
    with torch.cuda.graph(graph):
        out = feed_forward(x, *args[1:])
    for i in range(4):
        x.copy_(args[0] * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, feed_forward(x.clone(), *args[1:]))


@pytest.mark.gpu
def test_calls_at_once_on_two_streams(dev):
    """The operators share no memory: two streams that run them at the same time give what each gives alone."""
    jobs = [ff_inputs(dev, rows, 320) for rows in (16, 700)]
    wants = [feed_forward(*job) for job in jobs]
    streams = [torch.cuda.Stream(dev) for _ in jobs]
    torch.cuda.synchronize()
    gots = [[], []]
    for _ in range(20):
        for stream, job, got in zip(streams, jobs, gots):
            with torch.cuda.stream(stream):
                got.append(feed_forward(*job))
    torch.cuda.synchronize()
    for want, got in zip(wants, gots):
        assert all(torch.equal(y, want) for y in got)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [1, 129, 384, 385])
def test_linear_few_k_tiles_on_the_largest_tile(dev, k):
    """One to four k-tiles, fewer than the ring's stages and the scales' groups hold (sums of integers, exact in every kernel)."""
    gen = torch.Generator(device=dev).manual_seed(k)
    x = torch.randint(-3, 4, (4096, k), generator=gen, device=dev).float()
    w = torch.randint(-3, 4, (4090, k), generator=gen, device=dev).float()
    y = torch.mm(x.double(), w.double().t().contiguous())
    for xf, wf in PAIRS:
        xq, wq = mx.quantize(x, xf), mx.quantize(w, wf)
        assert torch.equal(mx.dequantize(xq), x) and torch.equal(mx.dequantize(wq), w)
        assert torch.equal(mx.linear(xq, wq, out_dtype=torch.float32).double(), y)
        assert torch.equal(mx.linear(xq, wq), y.bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("xf,wf", PAIRS, ids=["a8w4", "a4w4", "a8w8", "a4w8"])
@pytest.mark.parametrize("m,n,k", [(4000, 3700, 160), (4000, 3700, 4100), (4200, 4100, 200), (2050, 4200, 1400), (1100, 9000, 40)])
@pytest.mark.parametrize("activation,out", [(None, torch.bfloat16), ("geglu", "mxfp8"), ("quick_gelu", torch.float32)], ids=["bf16", "geglu-mx8", "gelu-f32"])
def test_linear_tiles_of_large_products(dev, xf, wf, m, n, k, activation, out):
    """Sizes at which the large tiles are taken, with ragged edges on all sides; 64-bit reference on the device."""
    gen = torch.Generator(device=dev).manual_seed(m)
    x = mx.quantize(torch.randn(m, k, generator=gen, device=dev), xf)
    w = mx.quantize(torch.randn(n, k, generator=gen, device=dev) / math.sqrt(k), wf)
    b = torch.randn(n, generator=gen, device=dev)
    res = torch.randn(m, n, generator=gen, device=dev).to(out) if out == torch.bfloat16 else None
    got = mx.linear(x, w, b, activation=activation, **(dict(out_format=out) if isinstance(out, str) else dict(out_dtype=out, residual=res)))
    got = mx.dequantize(got) if isinstance(out, str) else got
    xv, wv = mx.dequantize(x).double(), mx.dequantize(w).double()
    y = torch.mm(xv, wv.t().contiguous()) + b.double()
    size = torch.mm(xv.abs(), wv.abs().t().contiguous()) + b.double().abs()
    check_linear(y, size, k, got, activation, out, res, (xf, wf) != ("mxfp4", "mxfp4") and out != torch.float32)
