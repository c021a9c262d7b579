"""Cases that measure the microscaled (MX) operators and the norms that feed them.

Three operators, as a low-precision transformer block uses them next to the bf16 / fp32 kernels of this package:

* ``norm``    h = x + residual (rounded to the storage type), y = RMSNorm(h) or LayerNorm(h), y in the storage type or
              quantised to an MX format in the same pass;
* ``quant``   a matrix to an MX format and back to the values that it stands for;
* ``linear``  y = act(x W^T + bias) + residual with W in an MX format and x either in one or quantised within the call.

MX formats: blocks of 32 consecutive values of a row share the scale 2^e, e = floor(log2(max|v|)) - emax, held as the
byte e + 127 (255: the block holds an infinity or a NaN and stands for NaN); the values v / 2^e are rounded to nearest
even and saturated to e4m3 (``mxfp8``, emax 8, largest 448) or e2m1 (``mxfp4``, emax 2, largest 6, two to a byte, the
lower nibble first).  Rows are padded with zeros to a multiple of 128 values.

``own`` false: plain torch operations; true: the package's kernels.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EMAX = {"mxfp8": 8, "mxfp4": 2}
LARGEST = {"mxfp8": 448.0, "mxfp4": 6.0}
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LARGEST_NORM = 16384 * 8192      # values of the largest norm
LARGEST_QUANT = 65536 * 1280
LARGEST_LINEAR = 8192 ** 3       # multiplications of the largest product


# ---- cases ---------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token's residual stream through the norm in front of a quantised product: latency
        dict(name="rms 1x1280 bf16 mxfp8", op="norm", kind="rms", rows=1, c=1280, dtype="bf16", residual=True, out="mxfp8"),
        # fp32 residual stream of a 32x32 latent, normalised in place of a LayerNorm, no quantisation
        dict(name="rms 1024x1280 f32", op="norm", kind="rms", rows=1024, c=1280, dtype="f32", residual=True, out="same"),
        # text encoder: 16 prompts of 77 tokens, LayerNorm in front of the quantised projections
        dict(name="layer 1232x768 bf16 mxfp8", op="norm", kind="layer", rows=1232, c=768, dtype="bf16", residual=False, out="mxfp8"),
        # a long prefill of a wide model: the bandwidth-bound end
        dict(name="rms 16384x8192 bf16 mxfp8", op="norm", kind="rms", rows=16384, c=8192, dtype="bf16", residual=True, out="mxfp8"),
        # one prompt's context, quantised for the cross-attention's key / value projections
        dict(name="quant 77x768 bf16 mxfp8", op="quant", rows=77, k=768, dtype="bf16", fmt="mxfp8"),
        # rows that are neither whole blocks nor aligned
        dict(name="quant 1003x1283 f32 mxfp4", op="quant", rows=1003, k=1283, dtype="f32", fmt="mxfp4"),
        # gated feed-forward product of 16 64x64 latents
        dict(name="quant 65536x1280 bf16 mxfp4", op="quant", rows=65536, k=1280, dtype="bf16", fmt="mxfp4"),
        # a single row through a projection, quantised within the call: time embedding, one decoded token
        dict(name="linear 1x1280x1280 bf16", op="linear", m=1, n=1280, k=1280, x="mxfp8", w="mxfp4", given="plain", act="none", bias=True,
             residual=False, out="bf16"),
        # a small decode batch over wide weights: bound by reading them
        dict(name="linear 16x8192x8192 w4a8", op="linear", m=16, n=8192, k=8192, x="mxfp8", w="mxfp4", given="mx", act="none", bias=False,
             residual=True, out="bf16"),
        # nothing divides anything, fp32 result
        dict(name="linear 1001x1283x1000 w8a8", op="linear", m=1001, n=1283, k=1000, x="mxfp8", w="mxfp8", given="mx", act="none", bias=True,
             residual=True, out="f32"),
        # first half of a gated feed-forward at 16 64x64 latents, its product quantised for the second half
        dict(name="linear 65536x2560x320 geglu", op="linear", m=65536, n=2560, k=320, x="mxfp8", w="mxfp4", given="mx", act="geglu", bias=True,
             residual=False, out="mxfp8"),
        # the matrix-rate end: both sides in 4 bits
        dict(name="linear 8192x8192x8192 w4a4", op="linear", m=8192, n=8192, k=8192, x="mxfp4", w="mxfp4", given="mx", act="none", bias=False,
             residual=False, out="bf16"),
    ]


def _size(rng, low, high):
    """Spread over the logarithm; half of them rounded to a multiple of 64 where that leaves something."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and v >= 64:
        v -= v % 64
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(("norm", "quant", "linear", "linear"))
    if op == "norm":
        c = _size(rng, 8, 16384)
        rows = _size(rng, 1, max(1, min(65536, LARGEST_NORM // 2 // c)))
        return dict(op=op, kind=rng.choice(("rms", "rms", "layer")), rows=rows, c=c, dtype=rng.choice(("bf16", "f32")),
                    residual=rng.random() < 0.6, out=rng.choice(("same", "mxfp8", "mxfp8", "mxfp4")))
    if op == "quant":
        k = _size(rng, 8, 16384)
        rows = _size(rng, 1, max(1, min(65536, LARGEST_QUANT // 2 // k)))
        return dict(op=op, rows=rows, k=k, dtype=rng.choice(("bf16", "f32")), fmt=rng.choice(("mxfp8", "mxfp4")))
    n, k = _size(rng, 16, 8192), _size(rng, 32, 8192)
    m = _size(rng, 1, max(1, min(65536, LARGEST_LINEAR // 2 // (n * k), (1 << 27) // max(n, k))))
    act = rng.choice(("none", "none", "quick_gelu", "geglu"))
    if act == "geglu":
        n += n % 2
    x, w = rng.choice((("mxfp8", "mxfp4"), ("mxfp8", "mxfp4"), ("mxfp4", "mxfp4"), ("mxfp8", "mxfp8")))
    out = rng.choice(("bf16", "bf16", "f32", "mxfp8"))
    return dict(op=op, m=m, n=n, k=k, x=x, w=w, given=rng.choice(("mx", "plain")), act=act, bias=rng.random() < 0.7,
                residual=out in TYPES and rng.random() < 0.5, out=out)


def work(case):
    def mx(rows, k, fmt):
        return rows * k * {"mxfp8": 1.0, "mxfp4": 0.5}[fmt] + rows * -(-k // 32)

    size = {"bf16": 2, "f32": 4}
    if case["op"] == "norm":
        n, e = case["rows"] * case["c"], size[case["dtype"]]
        moved = n * e * (3 if case["residual"] else 1) + (n * e if case["out"] == "same" else mx(case["rows"], case["c"], case["out"]))
        return {"bytes": moved + 4 * case["c"], "flops": 6 * n}
    if case["op"] == "quant":
        n = case["rows"] * case["k"]
        return {"bytes": 2 * n * size[case["dtype"]] + mx(case["rows"], case["k"], case["fmt"]), "flops": 3 * n}
    m, n, k = case["m"], case["n"], case["k"]
    wide = n // 2 if case["act"] == "geglu" else n
    one = size[case["out"]] * m * wide if case["out"] in size else mx(m, wide, case["out"])
    moved = mx(m, k, case["x"]) if case["given"] == "mx" else 2 * m * k
    moved += mx(n, k, case["w"]) + one * (2 if case["residual"] else 1) + (4 * n if case["bias"] else 0)
    return {"bytes": moved, "flops": 2 * m * n * k}


# ---- inputs --------------------------------------------------------------------------------------------------------
def _activations(rows, c, dtype, gen):
    """Normal values; one channel in 64 is far wider than the others, as in the residual streams of transformers."""
    x = torch.randn(rows, c, generator=gen, device=DEVICE)
    wide = torch.rand(c, generator=gen, device=DEVICE) < 1 / 64
    return x.mul_(torch.where(wide, 24.0, 1.0)).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "norm":
        t, rows, c = TYPES[case["dtype"]], case["rows"], case["c"]
        s["x"] = _activations(rows, c, t, gen)
        s["residual"] = _activations(rows, c, t, gen) if case["residual"] else None
        s["weight"] = 1 + 0.2 * torch.randn(c, generator=gen, device=DEVICE)
        s["bias"] = 0.1 * torch.randn(c, generator=gen, device=DEVICE) if case["kind"] == "layer" else None
        return s
    if case["op"] == "quant":
        s["x"] = _activations(case["rows"], case["k"], TYPES[case["dtype"]], gen)
        return s
    m, n, k = case["m"], case["n"], case["k"]
    x = _activations(m, k, torch.bfloat16, gen)
    s["x"] = x if case["given"] == "plain" else _encode(x, case["x"])
    w = torch.randn(n, k, generator=gen, device=DEVICE) / math.sqrt(k)
    s["w"] = _encode(w, case["w"])  # what a program makes of its weights once and keeps
    wide = n // 2 if case["act"] == "geglu" else n
    s["bias"] = 0.1 * torch.randn(n, generator=gen, device=DEVICE) if case["bias"] else None
    s["residual"] = _activations(m, wide, TYPES[case["out"]], gen) if case["residual"] else None
    return s


# ---- the plain form ------------------------------------------------------------------------------------------------
def _power(e):
    """2^e exactly, for int32 e in [-127, 127] (-127 is a subnormal)."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).view(torch.float32)


def _blocks(v):
    rows, k = v.shape
    return torch.nn.functional.pad(v, (0, -k % 32)).view(rows, -1, 32)


def _quantised(v, fmt):
    """fp32 [rows, k] -> (values on the format's grid [rows, blocks, 32], exponents [rows, blocks], blocks that are NaN)."""
    b = _blocks(v)
    top = b.abs().amax(dim=2)
    bad = ~torch.isfinite(top)
    top = torch.where(bad, 0.0, top)
    e = torch.where(top > 0, torch.frexp(top)[1].int() - 1 - EMAX[fmt], -127).clamp(-127, 127)
    u = (b * _power(-e)[..., None]).clamp(-LARGEST[fmt], LARGEST[fmt])
    lowest, bits = (-6, 3) if fmt == "mxfp8" else (0, 1)  # least exponent, bits behind the point
    step = _power((torch.frexp(u)[1].int() - 1).clamp(min=lowest) - bits)
    return torch.where(bad[..., None], 0.0, torch.round(u / step) * step), e, bad


def _values(v, fmt):
    """The values that the quantised rows stand for, fp32 [rows, k]."""
    q, e, bad = _quantised(v, fmt)
    q = torch.where(bad[..., None], float("nan"), q * _power(e)[..., None])
    return q.view(v.shape[0], -1)[:, :v.shape[1]]


def _encode(v, fmt):
    """(codes, scales, k) in the layout that the module's docstring gives."""
    rows, k = v.shape
    q, e, bad = _quantised(v.float(), fmt)
    scales = torch.where(bad, 255, e + 127).to(torch.uint8)
    q = torch.nn.functional.pad(q.view(rows, -1), (0, -q.shape[1] * 32 % 128))
    scales = torch.nn.functional.pad(scales, (0, -scales.shape[1] % 4))
    if fmt == "mxfp8":
        codes = q.to(torch.float8_e4m3fn).view(torch.uint8)  # exact: q is on the grid
    else:
        grid = torch.tensor(FP4, device=v.device)
        code = torch.bucketize(q.abs(), grid) + 8 * torch.signbit(q)
        codes = (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8)
    return codes.contiguous(), scales.contiguous(), k


def _decode(t, fmt):
    codes, scales, k = t
    if fmt == "mxfp8":
        c = codes.int()
        exponent, fraction = (c >> 3) & 15, (c & 7).float()
        size = torch.where(exponent > 0, (8 + fraction) * _power(exponent - 10), fraction * 2.0 ** -9)
        size = torch.where((c & 127) == 127, float("nan"), size)
        v = torch.where(c > 127, -size, size)
    else:
        table = torch.tensor(FP4 + tuple(-x for x in FP4), device=codes.device)
        v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), dim=2)
    e = torch.where(scales < 255, _power(scales.int() - 127), float("nan"))
    return (v.view(codes.shape[0], -1, 32) * e[..., None]).view(codes.shape[0], -1)[:, :k]


def _plain_norm(s):
    case = s["case"]
    t = TYPES[case["dtype"]]
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(t)
    v = h.float()
    if case["kind"] == "rms":
        y = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + 1e-6) * s["weight"]
    else:
        d = v - v.mean(dim=1, keepdim=True)
        y = d / torch.sqrt((d * d).mean(dim=1, keepdim=True) + 1e-5) * s["weight"] + s["bias"]
    y = y.to(t) if case["out"] == "same" else _values(y, case["out"]).to(torch.bfloat16)
    return {"y": y} if s["residual"] is None else {"y": y, "h": h}


def _plain_linear(s):
    case = s["case"]
    x = _values(s["x"].float(), case["x"]) if case["given"] == "plain" else _decode(s["x"], case["x"])
    y = x @ _decode(s["w"], case["w"]).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["act"] == "quick_gelu":
        y = y / (1 + torch.exp(-1.702 * y))
    elif case["act"] == "geglu":
        v, g = y.chunk(2, dim=1)
        y = v * (0.5 * g * (1 + torch.erf(g * math.sqrt(0.5))))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(TYPES[case["out"]]) if case["out"] in TYPES else _values(y, case["out"]).to(torch.bfloat16)


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if own:
        return _own(s)
    if case["op"] == "norm":
        return _plain_norm(s)
    if case["op"] == "quant":
        return _values(s["x"].float(), case["fmt"]).to(s["x"].dtype)
    return _plain_linear(s)


def _own(s):
    from diffusion_model_amd import mx
    case = s["case"]
    if case["op"] == "norm":
        fmt = None if case["out"] == "same" else case["out"]
        if case["kind"] == "rms":
            y = mx.rmsnorm(s["x"], s["weight"], residual=s["residual"], eps=1e-6, out_format=fmt)
        else:
            y = mx.layernorm(s["x"], s["weight"], s["bias"], residual=s["residual"], eps=1e-5, out_format=fmt)
        y, h = y if s["residual"] is not None else (y, None)
        y = y if fmt is None else mx.dequantize(y, torch.bfloat16)
        return {"y": y} if h is None else {"y": y, "h": h}
    if case["op"] == "quant":
        return mx.dequantize(mx.quantize(s["x"], case["fmt"]), s["x"].dtype)
    x = s["x"] if case["given"] == "plain" else mx.MXTensor(*s["x"], case["x"])
    out = dict(out_dtype=TYPES[case["out"]]) if case["out"] in TYPES else dict(out_format=case["out"])
    y = mx.linear(x, mx.MXTensor(*s["w"], case["w"]), s["bias"], x_format=case["x"], activation=None if case["act"] == "none" else case["act"],
                  residual=s["residual"], **out)
    return y if case["out"] in TYPES else mx.dequantize(y, torch.bfloat16)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------
def _exact_values(v, fmt):
    """Nearest grid point by comparison with the midpoints between neighbours, in 64 bits, some rows at a time."""
    bits, lowest, highest = (3, -6, 8) if fmt == "mxfp8" else (1, 0, 2)
    grid = [i * 2.0 ** (lowest - bits) for i in range(1 << bits)]
    grid += [(1 + i / (1 << bits)) * 2.0 ** p for p in range(lowest, highest + 1) for i in range(1 << bits)]
    grid = torch.tensor([g for g in grid if g <= LARGEST[fmt]], dtype=torch.float64, device=v.device)
    middle = (grid[1:] + grid[:-1]) / 2
    out = torch.empty_like(v)
    chunk = max(1, (1 << 25) // max(1, v.shape[1]))
    for at in range(0, v.shape[0], chunk):
        x = v[at:at + chunk]
        b = _blocks(x)
        top = b.abs().amax(dim=2, keepdim=True)
        e = torch.floor(torch.log2(top.clamp(min=1e-300))) - EMAX[fmt]
        e = torch.where(torch.exp2(e + EMAX[fmt]) > top, e - 1, torch.where(torch.exp2(e + EMAX[fmt] + 1) <= top, e + 1, e))
        size = torch.exp2(e.clamp(min=-127, max=127))
        u = b.abs() / size
        below, above = torch.bucketize(u, middle), torch.bucketize(u, middle, right=True)
        pick = torch.where(below % 2 == 0, below, above)  # they differ on a midpoint alone: the even one of the two
        q = torch.sign(b) * grid[pick] * size
        out[at:at + chunk] = q.view(x.shape[0], -1)[:, :x.shape[1]]
    return out


def _exact_decode(t, fmt):
    codes, scales, k = t
    if fmt == "mxfp8":
        v = codes.view(torch.float8_e4m3fn).double()
    else:
        grid = torch.tensor(FP4, dtype=torch.float64, device=codes.device)
        nibbles = torch.stack((codes % 16, codes // 16), dim=-1).flatten(1).long()
        v = grid[nibbles % 8] * (1 - 2 * (nibbles // 8))
    return (v * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1))[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quant":
        return _exact_values(s["x"].double(), case["fmt"])
    if case["op"] == "norm":
        t = TYPES[case["dtype"]]
        h = s["x"] if s["residual"] is None else (s["x"].double() + s["residual"].double()).to(t)
        v = h.double()
        if case["kind"] == "layer":
            v = v - v.mean(dim=1, keepdim=True)
        y = v * torch.rsqrt(v.square().mean(dim=1, keepdim=True) + (1e-6 if case["kind"] == "rms" else 1e-5)) * s["weight"].double()
        if s["bias"] is not None:
            y = y + s["bias"].double()
        y = y if case["out"] == "same" else _exact_values(y, case["out"])
        return {"y": y} if s["residual"] is None else {"y": y, "h": h.double()}
    x = _exact_values(s["x"].double(), case["x"]) if case["given"] == "plain" else _exact_decode(s["x"], case["x"])
    y = torch.mm(x, _exact_decode(s["w"], case["w"]).t().contiguous())
    if s["bias"] is not None:
        y = y + s["bias"].double()
    if case["act"] == "quick_gelu":
        y = y * torch.sigmoid(1.702 * y)
    elif case["act"] == "geglu":
        wide = case["n"] // 2
        y = y[:, :wide] * torch.special.ndtr(y[:, wide:]) * y[:, wide:]
    if s["residual"] is not None:
        y = y + s["residual"].double()
    return y if case["out"] in TYPES else _exact_values(y, case["out"])
