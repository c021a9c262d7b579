"""Microscaled (MX) 8- and 4-bit operands for inference: quantisation, products, and the row norms that feed them.

    w = mx.quantize(linear.weight, "mxfp4")                        # once
    a, h = mx.rmsnorm(x, gamma, residual=h, out_format="mxfp8")    # h + x, its norm, quantised: one pass
    g = mx.linear(a, w, bias, activation="geglu", out_format="mxfp8")
    y = mx.linear(g, w2, bias2, residual=h)                        # bf16 rows

A matrix is quantised in blocks of 32 consecutive values of a row that share a power of two: ``mxfp8`` holds e4m3 values
(largest 448), ``mxfp4`` e2m1 values (largest 6, two to a byte).  A block's scale is 2^e with
e = floor(log2(largest magnitude)) - 8 (mxfp8) or - 2 (mxfp4), at least -127, stored as the byte e + 127; values are rounded to
nearest even and saturated.  A block that holds an infinity or a NaN stands for NaN (byte 255).

Matrices are 2-D row-major views ``[rows, k]`` with any row stride, as everywhere in this package; norm weights and biases are float32
whatever the rows' type; tensors live on the HIP device, results are new tensors, launches go to the current stream of the
operands' device.  Nothing here has a backward pass.
"""
from __future__ import annotations

from ctypes import byref
from typing import Optional

import torch

from . import _lib
from ._lib import MxGemmDesc, RowNormDesc, check
from .schedulers.base_scheduler import require_hip

FORMATS = {"mxfp8": _lib.DM_MXFP8, "mxfp4": _lib.DM_MXFP4}
_DTYPES = {torch.float32: _lib.DM_F32, torch.bfloat16: _lib.DM_BF16}
_ACTIVATIONS = {None: _lib.EPI_PLAIN, "quick_gelu": _lib.EPI_QUICKGELU, "geglu": _lib.EPI_GEGLU}
BLOCK, PAD, MAX_K = 32, 128, 1 << 24
MAX_ROWS, MAX_COLUMNS = 1 << 30, 1 << 24  # of a product


def _padded(k: int) -> int:
    return (k + PAD - 1) // PAD * PAD


class MXTensor:
    """A quantised matrix of ``rows`` rows of ``k`` values.

    ``codes``: uint8 ``[rows, kp]`` (mxfp8) or ``[rows, kp / 2]`` (mxfp4; the even value in the low nibble) with kp = k rounded
    up to 128 and zeros behind column k; ``scales``: uint8 ``[rows, kp / 32]``, anything behind the last block that holds values.  Both
    may have a row stride (a multiple of 16 and of 4 bytes).  Matrices quantised elsewhere in this format are wrapped as they are."""
    # Results of this module hold one buffer, codes then scales, and make the two views when somebody asks for them: an
    # allocation or a view costs a small call more than a microsecond each.
    __slots__ = ("_buffer", "_codes", "_scales", "rows", "k", "fmt", "device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, k: int, fmt: str):
        bits = _format(fmt)
        kp = _padded(k)
        if not 1 <= k <= MAX_K:
            raise ValueError(f"MXTensor: k must be between 1 and {MAX_K}, got {k}")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() != 2 or scales.dim() != 2:
            raise RuntimeError("MXTensor: codes and scales are 2-D uint8 tensors")
        (rows, width), shape = codes.shape, scales.shape
        if width != kp * bits // 8 or shape != (rows, kp // BLOCK):
            raise RuntimeError(f"MXTensor: {fmt} rows of {k} values are {kp * bits // 8} code and {kp // BLOCK} scale bytes, got "
                               f"{tuple(codes.shape)} and {tuple(shape)}")
        if codes.device != scales.device:
            raise RuntimeError(f"MXTensor: codes are on {codes.device}, scales on {scales.device}")
        self._buffer, self._codes, self._scales = None, codes, scales
        self.rows, self.k, self.fmt, self.device = rows, k, fmt, codes.device

    @classmethod
    def _empty(cls, rows: int, k: int, fmt: str, bits: int, device):
        """A new matrix and the four layout arguments of the C entry points: codes, bytes per row, scales, bytes per row."""
        kp = _padded(k)
        width, blocks = kp * bits // 8, kp // BLOCK
        t = cls.__new__(cls)
        t._buffer = torch.empty(rows * (width + blocks), dtype=torch.uint8, device=device)
        t._codes = t._scales = None
        t.rows, t.k, t.fmt, t.device = rows, k, fmt, device
        at = t._buffer.data_ptr()
        return t, at, width, at + rows * width, blocks

    def _layout(self, what: str):
        """The same four arguments of a matrix that is read."""
        buffer = self._buffer
        if buffer is not None:
            kp = _padded(self.k)
            width, at = kp * FORMATS[self.fmt] // 8, buffer.data_ptr()
            return at, width, at + self.rows * width, kp // BLOCK
        codes, scales = self._codes, self._scales
        if not codes.is_cuda:
            require_hip(codes, what)
        (ldc, one), (lds, also) = codes.stride(), scales.stride()
        if one != 1 or also != 1:
            raise RuntimeError(f"{what}: the bytes of a row of an MXTensor must be next to each other")
        if self.rows <= 1:  # torch gives a single row any stride
            ldc, lds = codes.shape[1], scales.shape[1]
        return codes.data_ptr(), ldc, scales.data_ptr(), lds

    def _view(self):
        n = self.rows * (_padded(self.k) * FORMATS[self.fmt] // 8)
        self._codes = self._buffer[:n].view(self.rows, _padded(self.k) * FORMATS[self.fmt] // 8)
        self._scales = self._buffer[n:].view(self.rows, _padded(self.k) // BLOCK)

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._view()
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._view()
        return self._scales

    @property
    def shape(self):
        return (self.rows, self.k)

    def __repr__(self) -> str:
        return f"MXTensor({self.rows} x {self.k}, {self.fmt}, {self.device})"


def _format(fmt: str) -> int:
    if fmt not in FORMATS:
        raise ValueError(f"unknown MX format {fmt!r}; expected one of {sorted(FORMATS)}")
    return FORMATS[fmt]


def _rows(t: torch.Tensor, what: str, name: str) -> None:
    """Refuses what the kernels do not read: they take 2-D rows on the device, a row's values next to each other."""
    if not t.is_cuda:
        require_hip(t, what)
    if t.dim() != 2:
        raise RuntimeError(f"{what}: {name} must be a 2-D matrix of rows, got {tuple(t.shape)}")
    if t.dtype not in _DTYPES:
        raise RuntimeError(f"{what}: {name} has dtype {t.dtype}; float32 or bfloat16 are supported")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise RuntimeError(f"{what}: the values of a row of {name} must be next to each other (stride {t.stride()})")


def _ld(t: torch.Tensor, rows: int, k: int) -> int:
    """Row stride in elements; torch gives a single row any stride."""
    return k if rows <= 1 else t.stride(0)


def _vector(t: Optional[torch.Tensor], n: int, device, what: str, name: str) -> Optional[int]:
    if t is None:
        return None
    if t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1) or t.device != device:
        raise RuntimeError(f"{what}: {name} must be {n} contiguous float32 values on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _check_width(k: int, what: str):
    if not 1 <= k <= MAX_K:
        raise ValueError(f"{what}: rows must have between 1 and {MAX_K} values, got {k}")


# The raw stream handle without a Stream object around it: a call here takes 5 to 9 us on the host, of which that was 2.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _call(fn, what: str, device: torch.device, *args):
    """One C entry point on the current stream of ``device``.  Launches go to the current device: make it that one meanwhile."""
    index = device.index
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        check(rc, what)


def quantize(x: torch.Tensor, fmt: str = "mxfp8") -> MXTensor:
    """fp32 / bf16 rows ``[rows, k]`` -> :class:`MXTensor`."""
    bits = _format(fmt)
    _rows(x, "mx.quantize", "x")
    rows, k = x.shape
    _check_width(k, "mx.quantize")
    device = x.device
    out, *layout = MXTensor._empty(rows, k, fmt, bits, device)
    _call(_lib.lib().dm_mx_quantize, "mx_quantize", device, x.data_ptr(), _ld(x, rows, k), rows, k, _DTYPES[x.dtype], bits, *layout)
    return out


def dequantize(t: MXTensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that ``t`` stands for, ``[rows, k]`` fp32 or bf16."""
    if dtype not in _DTYPES:
        raise RuntimeError(f"mx.dequantize: dtype {dtype} is not supported (float32 or bfloat16)")
    layout = t._layout("mx.dequantize")
    device, rows, k = t.device, t.rows, t.k
    out = torch.empty(rows, k, dtype=dtype, device=device)
    _call(_lib.lib().dm_mx_dequantize, "mx_dequantize", device, *layout, rows, k, FORMATS[t.fmt], out.data_ptr(), k, _DTYPES[dtype])
    return out


def _norm(what, kind, x, weight, bias, residual, eps, out_format):
    _rows(x, what, "x")
    rows, c = x.shape
    _check_width(c, what)
    device, dtype = x.device, x.dtype
    h, r_ptr, ldr, h_ptr = None, None, 0, None
    if residual is not None:
        _rows(residual, what, "residual")
        if residual.shape != x.shape or residual.dtype != dtype or residual.device != device:
            raise RuntimeError(f"{what}: residual must match x ({dtype} {tuple(x.shape)} on {device}), got {residual.dtype} "
                               f"{tuple(residual.shape)} on {residual.device}")
        h = torch.empty(rows, c, dtype=dtype, device=device)
        r_ptr, ldr, h_ptr = residual.data_ptr(), _ld(residual, rows, c), h.data_ptr()
    if out_format is None:
        y = torch.empty(rows, c, dtype=dtype, device=device)
        bits, y_ptr, ldy, ys_ptr, ldys = 0, y.data_ptr(), c, None, 0
    else:
        bits = _format(out_format)
        y, y_ptr, ldy, ys_ptr, ldys = MXTensor._empty(rows, c, out_format, bits, device)
    d = RowNormDesc(x.data_ptr(), _ld(x, rows, c), r_ptr, ldr, h_ptr, c, _vector(weight, c, device, what, "weight"),
                    _vector(bias, c, device, what, "bias"), y_ptr, ldy, ys_ptr, ldys, rows, c, _DTYPES[dtype], kind, bits, eps)
    _call(_lib.lib().dm_row_norm, "row_norm", device, byref(d))
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
    instructions, which lose about 2e-5 of an 8-bit product (where that matters, quantise or round an fp32 result).  fp32 results are fp32 sums of exact products, with activations right to a few
    units; for them an 8-bit operand's values are held in bf16, so those of scale bytes 0 to 2 are rounded to multiples of 2^-133 and those
    past bf16's largest (byte 247 on, which ``quantize`` never writes) are infinite."""
    what = "mx.linear"
    if activation not in _ACTIVATIONS:
        raise ValueError(f"{what}: unknown activation {activation!r}")
    if not isinstance(w, MXTensor):
        raise RuntimeError(f"{what}: w must be an MXTensor (mx.quantize)")
    x_src = _lib.X_MX
    if not isinstance(x, MXTensor):
        bits = _format(x_format)
        _rows(x, what, "x")
        if x.shape[0] <= _lib.X_ROWS_MAX_M:
            # few rows: the product quantises them itself as it reads them (1 x 1280 x 1280: one launch of two)
            x_src = _lib.X_BF16 if x.dtype == torch.bfloat16 else _lib.X_F32
            (m, k), device = x.shape, x.device
            x_ptr, ldx, xs_ptr, ld_xs = x.data_ptr(), _ld(x, m, k), None, 0
        else:
            x = quantize(x, x_format)
    if x_src == _lib.X_MX:
        bits, m, k, device = FORMATS[x.fmt], x.rows, x.k, x.device
        x_ptr, ldx, xs_ptr, ld_xs = x._layout(what)
    if k != w.k:
        raise RuntimeError(f"{what}: x has rows of {k} values, w of {w.k}")
    if device != w.device:
        raise RuntimeError(f"{what}: x is on {device}, w on {w.device}")
    n = w.rows
    if n < 1 or (activation == "geglu" and n % 2):
        raise RuntimeError(f"{what}: {n} output columns" + (" cannot be halved for geglu" if n else ""))
    if m > MAX_ROWS or n > MAX_COLUMNS:
        raise RuntimeError(f"{what}: a product of {m} x {n} is too large (at most {MAX_ROWS} x {MAX_COLUMNS})")
    wide = n // 2 if activation == "geglu" else n
    r_ptr, ldr, cs_ptr, ld_cs = None, 0, None, 0
    if out_format is None:
        if out_dtype not in _DTYPES:
            raise RuntimeError(f"{what}: out_dtype {out_dtype} is not supported (float32 or bfloat16)")
        y = torch.empty(m, wide, dtype=out_dtype, device=device)
        c_ptr, ldc, c_type = y.data_ptr(), wide, _DTYPES[out_dtype]
        if residual is not None:
            _rows(residual, what, "residual")
            if residual.shape != y.shape or residual.dtype != out_dtype or residual.device != device:
                raise RuntimeError(f"{what}: residual must match the result ({out_dtype} {tuple(y.shape)} on {device}), got "
                                   f"{residual.dtype} {tuple(residual.shape)} on {residual.device}")
            r_ptr, ldr = residual.data_ptr(), _ld(residual, m, wide)
    else:
        if residual is not None:
            raise RuntimeError(f"{what}: a quantised result takes no residual")
        c_type = _format(out_format)
        y, c_ptr, ldc, cs_ptr, ld_cs = MXTensor._empty(m, wide, out_format, c_type, device)
    d = MxGemmDesc(x_ptr, ldx, xs_ptr, ld_xs, *w._layout(what), bits, FORMATS[w.fmt], x_src, m, n, k, _vector(bias, n, device, what, "bias"),
                   r_ptr, ldr, c_ptr, ldc, cs_ptr, ld_cs, c_type, _ACTIVATIONS[activation])
    _call(_lib.lib().dm_mx_gemm, "mx_gemm", device, byref(d))
    return y
