"""Microscaled (MX) 8- and 4-bit operands for inference: quantisation, products, and the row norms that feed them.

    w = mx.quantize(linear.weight, "mxfp4")                        # once
    a, h = mx.rmsnorm(x, gamma, residual=h, out_format="mxfp8")    # h + x, its norm, quantised: one pass
    g = mx.linear(a, w, bias, activation="geglu", out_format="mxfp8")
    y = mx.linear(g, w2, bias2, residual=h)                        # bf16 rows

A matrix is quantised in blocks of 32 consecutive values of a row that share a power of two: ``mxfp8`` holds e4m3 values
(largest 448), ``mxfp4`` e2m1 values (largest 6, two to a byte).  A block's scale is 2^e with
e = floor(log2(largest magnitude)) - 8 (mxfp8) or - 2 (mxfp4), at least -127, stored as the byte e + 127; values are rounded to
nearest even and saturated.  A block that holds an infinity or a NaN stands for NaN (byte 255).

Matrices are 2-D row-major views ``[rows, k]`` with any row stride, as everywhere in this package; tensors live on the HIP
device, results are new tensors, launches go to the current stream of the operands' device.  Nothing here has a backward pass.
"""
from __future__ import annotations

from ctypes import byref
from typing import Optional

import torch

from . import _lib
from ._lib import MxGemmDesc, RowNormDesc, check
from .schedulers.base_scheduler import require_hip, stream_of

FORMATS = {"mxfp8": _lib.DM_MXFP8, "mxfp4": _lib.DM_MXFP4}
_DTYPES = {torch.float32: _lib.DM_F32, torch.bfloat16: _lib.DM_BF16}
_ACTIVATIONS = {None: _lib.EPI_PLAIN, "quick_gelu": _lib.EPI_QUICKGELU, "geglu": _lib.EPI_GEGLU}
BLOCK, PAD, MAX_K = 32, 128, 1 << 24


def _padded(k: int) -> int:
    return (k + PAD - 1) // PAD * PAD


class MXTensor:
    """A quantised matrix of ``rows`` rows of ``k`` values.

    ``codes``: uint8 ``[rows, kp]`` (mxfp8) or ``[rows, kp / 2]`` (mxfp4; the even value in the low nibble) with kp = k rounded
    up to 128 and zeros behind column k; ``scales``: uint8 ``[rows, kp / 32]``.  Both may have a row stride (a multiple of 16 and
    of 4 bytes).  Matrices quantised elsewhere in this format are wrapped as they are."""
    __slots__ = ("codes", "scales", "k", "fmt")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, k: int, fmt: str):
        bits = _format(fmt)
        kp = _padded(k)
        if not 1 <= k <= MAX_K:
            raise ValueError(f"MXTensor: k must be between 1 and {MAX_K}, got {k}")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() != 2 or scales.dim() != 2:
            raise RuntimeError("MXTensor: codes and scales are 2-D uint8 tensors")
        rows = codes.shape[0]
        if codes.shape[1] != kp * bits // 8 or scales.shape != (rows, kp // BLOCK):
            raise RuntimeError(f"MXTensor: {fmt} rows of {k} values are {kp * bits // 8} code and {kp // BLOCK} scale bytes, got "
                               f"{tuple(codes.shape)} and {tuple(scales.shape)}")
        if codes.device != scales.device:
            raise RuntimeError(f"MXTensor: codes are on {codes.device}, scales on {scales.device}")
        self.codes, self.scales, self.k, self.fmt = codes, scales, k, fmt

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    @property
    def shape(self):
        return (self.codes.shape[0], self.k)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def __repr__(self) -> str:
        return f"MXTensor({self.rows} x {self.k}, {self.fmt}, {self.codes.device})"


def _format(fmt: str) -> int:
    if fmt not in FORMATS:
        raise ValueError(f"unknown MX format {fmt!r}; expected one of {sorted(FORMATS)}")
    return FORMATS[fmt]


def _new(rows: int, k: int, fmt: str, device) -> MXTensor:
    kp = _padded(k)
    t = MXTensor.__new__(MXTensor)
    t.codes = torch.empty(rows, kp * FORMATS[fmt] // 8, dtype=torch.uint8, device=device)
    t.scales = torch.empty(rows, kp // BLOCK, dtype=torch.uint8, device=device)
    t.k, t.fmt = k, fmt
    return t


def _rows(t: torch.Tensor, what: str, name: str) -> torch.Tensor:
    """``t`` as the kernels read it: 2-D rows on the device, values next to each other (a single row may have any stride)."""
    if t.device.type != "cuda":
        require_hip(t, what)
    if t.dim() != 2:
        raise RuntimeError(f"{what}: {name} must be a 2-D matrix of rows, got {tuple(t.shape)}")
    if t.dtype not in _DTYPES:
        raise RuntimeError(f"{what}: {name} has dtype {t.dtype}; float32 or bfloat16 are supported")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise RuntimeError(f"{what}: the values of a row of {name} must be next to each other (stride {t.stride()})")
    return t


def _ld(t: torch.Tensor) -> int:
    """Row stride; torch gives a single row any stride, and an expanded one 0."""
    return max(t.stride(0), t.shape[1]) if t.shape[0] <= 1 else t.stride(0)


def _vector(t: Optional[torch.Tensor], n: int, device, what: str, name: str) -> Optional[int]:
    if t is None:
        return None
    if t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1) or t.device != device:
        raise RuntimeError(f"{what}: {name} must be {n} contiguous float32 values on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _check_width(k: int, what: str):
    if not 1 <= k <= MAX_K:
        raise ValueError(f"{what}: rows must have between 1 and {MAX_K} values, got {k}")


class _On:
    """Kernel launches go to the current device: make it the operands' one for the call."""
    __slots__ = ("index", "before")

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def quantize(x: torch.Tensor, fmt: str = "mxfp8") -> MXTensor:
    """fp32 / bf16 rows ``[rows, k]`` -> :class:`MXTensor`."""
    bits = _format(fmt)
    _rows(x, "mx.quantize", "x")
    rows, k = x.shape
    _check_width(k, "mx.quantize")
    out = _new(rows, k, fmt, x.device)
    with _On(x.device):
        check(_lib.lib().dm_mx_quantize(x.data_ptr(), _ld(x), rows, k, _DTYPES[x.dtype], bits, out.codes.data_ptr(), out.codes.shape[1],
                                        out.scales.data_ptr(), out.scales.shape[1], stream_of(x)), "mx_quantize")
    return out


def _operand(t: MXTensor, what: str):
    """(codes, row bytes, scales, row bytes) for the C entry points."""
    if t.codes.device.type != "cuda":
        require_hip(t.codes, what)
    if t.codes.stride(1) != 1 or (t.scales.shape[1] > 1 and t.scales.stride(1) != 1):
        raise RuntimeError(f"{what}: the bytes of a row of an MXTensor must be next to each other")
    return t.codes.data_ptr(), _ld(t.codes), t.scales.data_ptr(), _ld(t.scales)


def dequantize(t: MXTensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that ``t`` stands for, ``[rows, k]`` fp32 or bf16."""
    if dtype not in _DTYPES:
        raise RuntimeError(f"mx.dequantize: dtype {dtype} is not supported (float32 or bfloat16)")
    codes, ldc, scales, lds = _operand(t, "mx.dequantize")
    out = torch.empty(t.rows, t.k, dtype=dtype, device=t.device)
    with _On(t.device):
        check(_lib.lib().dm_mx_dequantize(codes, ldc, scales, lds, t.rows, t.k, FORMATS[t.fmt], out.data_ptr(), t.k, _DTYPES[dtype],
                                          stream_of(out)), "mx_dequantize")
    return out


def _norm(what, kind, x, weight, bias, residual, eps, out_format):
    _rows(x, what, "x")
    rows, c = x.shape
    _check_width(c, what)
    d = RowNormDesc(x=x.data_ptr(), ldx=_ld(x), gamma=_vector(weight, c, x.device, what, "weight"), beta=_vector(bias, c, x.device, what, "bias"),
                    rows=rows, c=c, dtype=_DTYPES[x.dtype], kind=kind, eps=eps)
    h = None
    if residual is not None:
        _rows(residual, what, "residual")
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise RuntimeError(f"{what}: residual must match x ({x.dtype} {tuple(x.shape)} on {x.device}), got {residual.dtype} "
                               f"{tuple(residual.shape)} on {residual.device}")
        h = torch.empty(rows, c, dtype=x.dtype, device=x.device)
        d.r, d.ldr, d.h, d.ldh = residual.data_ptr(), _ld(residual), h.data_ptr(), c
    if out_format is None:
        y = torch.empty(rows, c, dtype=x.dtype, device=x.device)
        d.y, d.ldy = y.data_ptr(), c
    else:
        d.out_fmt = _format(out_format)
        y = _new(rows, c, out_format, x.device)
        d.y, d.ldy, d.y_scales, d.ldys = y.codes.data_ptr(), y.codes.shape[1], y.scales.data_ptr(), y.scales.shape[1]
    with _On(x.device):
        check(_lib.lib().dm_row_norm(byref(d), stream_of(x)), "row_norm")
    return y if h is None else (y, h)


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
            out_format: Optional[str] = None):
    """``h / sqrt(mean(h^2) + eps) * weight`` over the rows of ``h = x + residual`` (rounded to x's type).

    Returns the normed rows in x's type, or an :class:`MXTensor` with ``out_format``; with ``residual`` a pair of it and ``h``."""
    return _norm("mx.rmsnorm", _lib.NORM_RMS, x, weight, None, residual, eps, out_format)


def layernorm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
              eps: float = 1e-5, out_format: Optional[str] = None):
    """``(h - mean(h)) / sqrt(var(h) + eps) * weight + bias``; otherwise as :func:`rmsnorm`."""
    return _norm("mx.layernorm", _lib.NORM_LAYER, x, weight, bias, residual, eps, out_format)


def linear(x, w: MXTensor, bias: Optional[torch.Tensor] = None, *, x_format: str = "mxfp8", activation: Optional[str] = None,
           residual: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16, out_format: Optional[str] = None):
    """``act(x w^T + bias) + residual``: x ``[m, k]`` (an :class:`MXTensor`, or fp32 / bf16 rows that are quantised to ``x_format``
    first), w ``[n, k]``, bias ``[n]`` float32.

    ``activation``: None, ``"quick_gelu"`` (v sigmoid(1.702 v)) or ``"geglu"`` (the first n / 2 columns times gelu(the others):
    ``[m, n / 2]``).  The result has ``out_dtype`` (bfloat16 / float32; ``residual`` has the same type), or is an
    :class:`MXTensor` with ``out_format`` (no residual).  Accumulation is fp32; bf16 and MX results come from the scaled matrix
    instructions, which lose about 2e-5 of an 8-bit product, fp32 results are exact to fp32."""
    what = "mx.linear"
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{what}: unknown activation {activation!r}")
    if not isinstance(w, MXTensor):
        raise RuntimeError(f"{what}: w must be an MXTensor (mx.quantize)")
    if not isinstance(x, MXTensor):
        x = quantize(x, x_format)
    if x.k != w.k:
        raise RuntimeError(f"{what}: x has rows of {x.k} values, w of {w.k}")
    if x.device != w.device:
        raise RuntimeError(f"{what}: x is on {x.device}, w on {w.device}")
    m, n, device = x.rows, w.rows, x.device
    if n < 1 or (activation == "geglu" and n % 2):
        raise RuntimeError(f"{what}: {n} output columns" + (" cannot be halved for geglu" if n else ""))
    wide = n // 2 if activation == "geglu" else n
    d = MxGemmDesc()
    d.x, d.ldx, d.x_scales, d.ld_xs = _operand(x, what)
    d.w, d.ldw, d.w_scales, d.ld_ws = _operand(w, what)
    d.x_fmt, d.w_fmt, d.m, d.n, d.k, d.epi = FORMATS[x.fmt], FORMATS[w.fmt], m, n, x.k, _ACTIVATIONS[activation]
    d.bias = _vector(bias, n, device, what, "bias")
    if out_format is None:
        if out_dtype not in _DTYPES:
            raise RuntimeError(f"{what}: out_dtype {out_dtype} is not supported (float32 or bfloat16)")
        y = torch.empty(m, wide, dtype=out_dtype, device=device)
        d.c, d.ldc, d.c_type = y.data_ptr(), wide, _DTYPES[out_dtype]
        if residual is not None:
            _rows(residual, what, "residual")
            if residual.shape != y.shape or residual.dtype != out_dtype or residual.device != device:
                raise RuntimeError(f"{what}: residual must match the result ({out_dtype} {tuple(y.shape)} on {device}), got "
                                   f"{residual.dtype} {tuple(residual.shape)} on {residual.device}")
            d.r, d.ldr = residual.data_ptr(), _ld(residual)
    else:
        if residual is not None:
            raise RuntimeError(f"{what}: a quantised result takes no residual")
        d.c_type = _format(out_format)
        y = _new(m, wide, out_format, device)
        d.c, d.ldc, d.c_scales, d.ld_cs = y.codes.data_ptr(), y.codes.shape[1], y.scales.data_ptr(), y.scales.shape[1]
    with _On(device):
        check(_lib.lib().dm_mx_gemm(byref(d), torch.cuda.current_stream(device).cuda_stream), "mx_gemm")
    return y
