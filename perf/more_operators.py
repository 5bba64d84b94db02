"""The feed-forward half of a layer on microscaled rows: the norm that makes them,
their quantisation, the product with 4 bit weights, the gated projections, and
the three in a row.

Microscaled rows: 32 consecutive values of a row share a power of two 2^e, one
byte e + 127 per block, and each value is a code times 2^e.  "e2m1": 4 bit codes
(0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte, the first in the low half;
"e4m3": 8 bit codes up to 448.  e is the smallest that keeps the block's largest
magnitude within the largest code, at least -126; codes are to nearest, ties to even.

Kinds of case (a case is a dict of plain values):

  norm      x + residual (the new residual stream, in its own type), its
            root-mean-square norm with a gain, quantised.
  quantize  rows quantised: a weight at load time, activations.
  matmul    weights [rows][cols] in 4 bits times activations [n][cols] in 8 or
            4, with a residual, f32 or bf16 out.
  gated     act(x Wg') * (x Wu'), quantised.
  block     norm, gated, matmul with the residual: a layer's feed-forward.

What is held in codes comes back as the values it stands for, in bf16, which
holds all of them exactly.
"""
from __future__ import annotations

import math
import pathlib
import sys

import torch

own = False

EPS = 1e-5


def _case(op, n, cols, rows=0, io="f32", act="e4m3", fn="silu"):
    """rows: the weight's; io: type of the rows that are not codes; act: codes of
    the activations (norm, quantize, gated: of the output too); fn: the gated
    block's activation."""
    return {"op": op, "n": n, "cols": cols, "rows": rows, "io": io, "act": act, "fn": fn}


# ------------------------------------------------------------------ cases


def listed():
    return [
        # a single position's norm: latency alone
        dict(_case("norm", 1, 4096), name="norm_one"),
        # the norm of a prompt's first pass, a bf16 stream
        dict(_case("norm", 8191, 3584, io="bf16"), name="norm_prompt"),
        # the scattered rows of a late denoise step, 4 bit activations
        dict(_case("quantize", 181, 2048, act="e2m1"), name="quantize_rows"),
        # a weight brought to 4 bits when a model is loaded
        dict(_case("quantize", 18944, 3584, io="bf16", act="e2m1"), name="quantize_weight"),
        # the down projection of a single position
        dict(_case("matmul", 1, 12288, 4096), name="matmul_one"),
        # a canvas's rows times a square projection, the f32 residual stream
        dict(_case("matmul", 256, 4096, 4096), name="matmul_canvas"),
        # a prompt's first pass, 8 bit activations
        dict(_case("matmul", 4096, 12288, 4096, io="bf16"), name="matmul_prompt"),
        # the same with 4 bit activations, a ragged number of rows
        dict(_case("matmul", 2553, 3584, 18944, io="bf16", act="e2m1"), name="matmul_prompt_4bit"),
        # one position through the gated projections
        dict(_case("gated", 1, 4096, 12288), name="gated_one"),
        # a prompt's first pass through them, gelu
        dict(_case("gated", 4096, 4096, 12288, fn="gelu"), name="gated_prompt"),
        # a layer's whole feed-forward for one position
        dict(_case("block", 1, 3584, 18944, io="bf16"), name="block_one"),
        # and for a denoise step's canvas
        dict(_case("block", 256, 4096, 12288, io="bf16"), name="block_canvas"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {n: max(work(c)[n] for c in listed()) for n in ("bytes", "flops")}
    while True:
        op = rng.choice(["norm", "quantize", "matmul", "matmul", "gated", "block"])
        n = rng.choice([rng.randint(1, 16), _log(rng, 1, 8192), _log(rng, 17, 600)])
        cols = 32 * _log(rng, 1, 448)
        rows = 0 if op in ("norm", "quantize") else _log(rng, 1, 19000) if op == "matmul" else 32 * _log(rng, 1, 592)
        c = _case(op, n, cols, rows, "bf16" if op == "block" else rng.choice(["f32", "bf16"]), rng.choice(["e4m3", "e4m3", "e2m1"]),
                  rng.choice(["silu", "gelu"]) if op in ("gated", "block") else "silu")
        w = work(c)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return c


def work(case):
    op, n, k, m = case["op"], case["n"], case["cols"], case["rows"]
    b = 4 if case["io"] == "f32" else 2
    code = (32 if case["act"] == "e4m3" else 16) / 32 + 1 / 32  # an activation's bytes
    w = 17 / 32  # a weight's
    if op == "norm":
        return {"bytes": 3 * n * k * b + 4 * k + n * k * code, "flops": 0}
    if op == "quantize":
        return {"bytes": n * k * (b + code), "flops": 0}
    if op == "matmul":
        return {"bytes": m * k * w + n * k * code + 2 * n * m * b, "flops": 2 * n * m * k}
    if op == "gated":
        return {"bytes": 2 * m * k * w + n * k * code + n * m * code, "flops": 4 * n * m * k}
    return {"bytes": 3 * m * k * w + 4 * k + n * k * b * 3, "flops": 6 * n * m * k}  # block: x, residual, out


# ------------------------------------------------------------------ inputs


def _type(case):
    return torch.float32 if case["io"] == "f32" else torch.bfloat16


def _inputs(case, seed):
    """Rows and weights on the GPU, f32 or the case's type.  Activations have
    channels of unequal size with a few far larger ones, as behind a norm's gain;
    weights rows of unequal size."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    op, n, k, m = case["op"], case["n"], case["cols"], case["rows"]
    t = _type(case)
    gain = torch.exp(0.5 * randn(k)) * (1 + 15 * (torch.rand(k, device="cuda", generator=gen) < 0.004).float())

    def weight(rows, cols):
        return randn(rows, cols) * torch.exp(0.3 * randn(rows, 1)) / math.sqrt(cols)

    s = {}
    if op in ("norm", "block"):
        s["x"], s["residual"] = randn(n, k).to(t), (randn(n, k) * torch.exp(0.3 * randn(k))).to(t)
        s["gain"] = gain
    elif op == "quantize":
        s["x"] = (randn(n, k) * gain).to(t)
    else:
        s["x"] = randn(n, k) * gain  # in codes before the call
    if op == "matmul":
        s["w"] = weight(m, k)
        s["residual"] = randn(n, m).to(t)
    if op in ("gated", "block"):
        s["gate"], s["up"] = weight(m, k), weight(m, k)
    if op == "block":
        s["down"] = weight(k, m)
    return s


def prepare(case, seed):
    """What a program holds before the call: rows, weights in 4 bit codes,
    and (matmul, gated) the activations in codes."""
    s = {"case": case, **_inputs(case, seed)}
    op, n, k, m = case["op"], case["n"], case["cols"], case["rows"]
    for name in ("w", "gate", "up", "down"):
        if name in s:
            s[name] = _quantise(s[name], "e2m1")
    if op in ("matmul", "gated"):
        s["x"] = _quantise(s["x"], case["act"])
    if own:
        dr, ctx = _framework()
        s["dr"], s["ctx"] = dr, ctx
        for name in ("w", "gate", "up", "down", "x"):
            if isinstance(s.get(name), tuple):
                s[name] = _rows(dr, "e2m1" if name != "x" else case["act"], *s[name])
        if op in ("norm", "quantize", "block"):
            s["codes"] = _empty(dr, case["act"], n, k)
        if op in ("norm", "quantize"):
            s["values"] = torch.empty(n, k, dtype=torch.bfloat16, device="cuda")
        if op in ("norm", "block"):
            s["sum"] = torch.empty_like(s["x"])
        if op in ("gated", "block"):
            s["hidden"] = _empty(dr, case["act"], n, m)
        if op == "gated":
            s["values"] = torch.empty(n, m, dtype=torch.bfloat16, device="cuda")
        if op == "matmul":
            s["out"] = torch.empty_like(s["residual"])
        if op == "block":
            s["out"] = torch.empty_like(s["x"])
    return s


_FRAMEWORK = []


def _framework():
    """The framework's module and a program's context."""
    if not _FRAMEWORK:
        path = str(pathlib.Path(__file__).resolve().parent.parent / "diffuse-rs_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import dr_attn as dr

        ctx, stream = dr.Context(torch.cuda.current_device()), torch.cuda.Stream()
        ctx.set_stream(stream.cuda_stream)
        _FRAMEWORK.extend([dr, ctx, stream])
    return _FRAMEWORK[:2]


def _format(dr, name):
    return dr.MX_E4M3 if name == "e4m3" else dr.MX_E2M1


def _pitch(cols):
    """Scale bytes of a row: one per 32 values, rows at multiples of 4 bytes."""
    return (cols // 32 + 3) // 4 * 4


def _rows(dr, fmt, codes, scales):
    n, blocks = scales.shape
    padded = torch.zeros(n, _pitch(32 * blocks), dtype=torch.uint8, device="cuda")
    padded[:, :blocks] = scales
    return dr.MxRows(codes, padded, _format(dr, fmt))


def _empty(dr, fmt, n, cols):
    codes = torch.empty(n, cols if fmt == "e4m3" else cols // 2, dtype=torch.uint8, device="cuda")
    return dr.MxRows(codes, torch.empty(n, _pitch(cols), dtype=torch.uint8, device="cuda"), _format(dr, fmt))


# ------------------------------------------------------------------ the operators


def run(s):
    case = s["case"]
    op, n, k, m = case["op"], case["n"], case["cols"], case["rows"]
    if not own:
        return _plain(case, s)
    dr, ctx = s["dr"], s["ctx"]
    dtype = dr.DTYPE_F32 if case["io"] == "f32" else dr.DTYPE_BF16
    fn = dr.ACT_SILU if case["fn"] == "silu" else dr.ACT_GELU
    if op == "norm":
        dr.rms_norm_mx(ctx, s["x"], n, k, s["codes"], w=s["gain"], eps=EPS, residual=s["residual"], total=s["sum"], dtype=dtype)
        dr.mx_dequantize(ctx, s["codes"], n, k, s["values"], dtype=dr.DTYPE_BF16)
        return [s["sum"], s["values"]]
    if op == "quantize":
        dr.mx_quantize(ctx, s["x"], n, k, s["codes"], dtype=dtype)
        dr.mx_dequantize(ctx, s["codes"], n, k, s["values"], dtype=dr.DTYPE_BF16)
        return s["values"]
    if op == "matmul":
        dr.mx_matmul(ctx, s["w"], m, k, s["x"], n, s["out"], residual=s["residual"], dtype=dtype)
        return s["out"]
    if op == "gated":
        dr.mx_gated(ctx, s["gate"], s["up"], m, k, s["x"], n, s["hidden"], activation=fn)
        dr.mx_dequantize(ctx, s["hidden"], n, m, s["values"], dtype=dr.DTYPE_BF16)
        return s["values"]
    dr.rms_norm_mx(ctx, s["x"], n, k, s["codes"], w=s["gain"], eps=EPS, residual=s["residual"], total=s["sum"], dtype=dtype)
    dr.mx_gated(ctx, s["gate"], s["up"], m, k, s["codes"], n, s["hidden"], activation=fn)
    dr.mx_matmul(ctx, s["down"], k, m, s["hidden"], n, s["out"], residual=s["sum"], dtype=dtype)
    return [s["sum"], s["out"]]


TOP = {"e2m1": (2, 0.75), "e4m3": (8, 0.875)}  # the largest code: exponent, half its mantissa (6 = 0.75 * 8, 448 = 0.875 * 512)


def _quantise(x, fmt):
    """Codes and scale bytes of rows [n, cols]."""
    n, cols = x.shape
    x = x.float().reshape(n, cols // 32, 32)
    big, half = TOP[fmt]
    mant, e = torch.frexp(x.abs().amax(-1, keepdim=True))  # amax = mant 2^e, mant in [0.5, 1)
    e = torch.clamp(e - 1 - big + (mant > half).to(torch.int32), min=-126)
    y = torch.ldexp(x, -e)
    scales = (e + 127).to(torch.uint8).reshape(n, cols // 32)
    if fmt == "e4m3":
        return y.to(torch.float8_e4m3fn).view(torch.uint8).reshape(n, cols), scales
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
            + 8 * torch.signbit(y)).reshape(n, cols // 2, 2)
    return code[..., 0] + 16 * code[..., 1], scales


def _values(codes, scales, fmt):
    """The f32 values that codes [n, ...] with scale bytes [n, blocks] stand for."""
    n, blocks = scales.shape
    if fmt == "e4m3":
        y = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
        y = table[torch.stack((codes & 15, codes >> 4), -1).int()]
    return torch.ldexp(y.reshape(n, blocks, 32), scales.to(torch.int32)[..., None] - 127).reshape(n, 32 * blocks)


def _act(x, fn):
    if fn == "silu":
        return x / (1 + torch.exp(-x))
    # 0.5 (1 + tanh z) = 1 / (1 + e^-2z), which keeps its digits where tanh is near -1
    return x / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))


def _plain(case, s):
    """The operators in elementary operations, 32 bits."""
    op, t, fmt = case["op"], _type(case), case["act"]
    if op in ("norm", "block"):
        h = (s["x"].float() + s["residual"].float()).to(t)
        f = h.float()
        y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * s["gain"]
        x = _quantise(y, fmt)
        if op == "norm":
            return [h, _values(*x, fmt).bfloat16()]
    elif op == "quantize":
        return _values(*_quantise(s["x"], fmt), fmt).bfloat16()
    else:
        x = s["x"]
    a = _values(*x, fmt)
    if op == "matmul":
        return (torch.matmul(a, _values(*s["w"], "e2m1").t()) + s["residual"].float()).to(t)
    hidden = _act(torch.matmul(a, _values(*s["gate"], "e2m1").t()), case["fn"]) * torch.matmul(a, _values(*s["up"], "e2m1").t())
    hidden = _quantise(hidden, fmt)
    if op == "gated":
        return _values(*hidden, fmt).bfloat16()
    return [h, (torch.matmul(_values(*hidden, fmt), _values(*s["down"], "e2m1").t()) + h.float()).to(t)]


# ------------------------------------------------------------------ the definition, in 64 bits


def _rounded(x, fmt):
    """The f64 values that rows x stand for once quantised."""
    shape = x.shape
    x = x.double().reshape(shape[0], shape[1] // 32, 32)
    largest, top, low, bits = (6.0, 2, 0, 1) if fmt == "e2m1" else (448.0, 8, -6, 3)
    most = x.abs().amax(-1, keepdim=True)
    unit = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(most, min=2.0**-140))) - top - 1, min=-126.0))
    unit = torch.where(most > largest * unit, 2 * unit, unit)  # from one or two below the answer upwards
    unit = torch.where(most > largest * unit, 2 * unit, unit)
    y = x / unit
    mag = torch.clamp(y.abs(), min=2.0**low)
    g = torch.floor(torch.log2(mag))
    g = torch.where(torch.exp2(g) > mag, g - 1, torch.where(torch.exp2(g + 1) <= mag, g + 1, g))
    step = torch.exp2(g - bits)
    return (torch.round(y / step) * step * unit).reshape(shape)  # (torch.round: half to even)


def exact(case, seed):
    s, op, t, fmt = _inputs(case, seed), case["op"], _type(case), case["act"]

    def product(a, w):
        return a @ _rounded(w, "e2m1").t().contiguous()

    if op in ("norm", "block"):
        h = (s["x"].double() + s["residual"].double()).float().to(t).double()  # the stream is held in its type
        y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS) * s["gain"].double()
        a = _rounded(y, fmt)
        if op == "norm":
            return [h, a]
    else:
        a = _rounded(s["x"], fmt)
        if op == "quantize":
            return a
    if op == "matmul":
        return product(a, s["w"]) + s["residual"].double()
    g = product(a, s["gate"])
    if case["fn"] == "silu":
        g = g * torch.special.expit(g)
    else:
        g = g * torch.special.expit(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g**3))  # (1 + tanh z) / 2 = 1 / (1 + e^-2z)
    hidden = _rounded(g * product(a, s["up"]), fmt)
    return hidden if op == "gated" else [h, product(hidden, s["down"]) + h]
