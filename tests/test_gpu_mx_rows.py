"""dr_mx_quantize, dr_mx_dequantize and dr_rms_norm_mx against tests/mx_reference.py
(64 bits).  Quantisation and reading back are exact; a norm's values are f32
sums, so its codes are those of some value within dy of the exact one:

  dy = |y| ((cols / 2048 + 2) 8 + 20) 2^-24

a thread of 256 adds up to cols / 256 squares one after the other (half of the
sum's relative error reaches the root; in longer rows a thread of 1024 adds by
eights), six lane exchanges, four partial sums, and eight roundings from there
to y.  Needs an MI355X."""
from __future__ import annotations

import numpy as np
import pytest

import dr_attn as dr
import mx_reference as mx
from test_gpu_parity import dev, say, torch  # noqa: F401

pytestmark = pytest.mark.gpu

FMTS = {"e2m1": dr.MX_E2M1, "e4m3": dr.MX_E4M3}
FILL = 0xA5


def put(dev, x, bf16=False):
    """f32 values (bf16-exact ones as bf16 bits) on the device."""
    if bf16:
        return dev.put((np.ascontiguousarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16).view(np.int16))
    return dev.put(np.ascontiguousarray(x, np.float32))


def get(dev, t, bf16=False):
    x = dev.get(t)
    return (x.view(np.uint16).astype(np.uint32) << 16).view(np.float32) if bf16 else x


def empty_rows(dev, n, cols, fmt, extra=64):
    """Rows with `extra` bytes behind each plane, all FILL."""
    codes = dev.put(np.full(n * (cols // 2 if fmt == dr.MX_E2M1 else cols) + extra, FILL, np.uint8))
    return dr.MxRows(codes, dev.put(np.full(n * dr.mx_pitch(cols) + extra, FILL, np.uint8)), fmt)


def put_rows(dev, codes, scales, fmt):
    return dr.MxRows(dev.put(codes), dev.put(scales), fmt)


def get_rows(dev, r, n, cols):
    """(codes, scales) of rows made by empty_rows; the bytes behind them and
    between their scales must be as they were."""
    w = cols // 2 if r.format == dr.MX_E2M1 else cols
    codes, scales = dev.get(r.codes), dev.get(r.scales)
    assert (codes[n * w:] == FILL).all() and (scales[n * dr.mx_pitch(cols):] == FILL).all()
    scales = scales[: n * dr.mx_pitch(cols)].reshape(n, -1)
    assert (scales[:, cols // 32:] == FILL).all()
    return codes[: n * w].reshape(n, w), scales


def rows_of_all_kinds(rng, n, cols, bf16):
    """Values of every size, zeros, ties, denormals, NaN and infinities."""
    x = rng.standard_normal((n, cols)) * np.exp2(rng.integers(-40, 40, (n, cols // 32))).repeat(32, axis=1)
    with np.errstate(over="ignore"):
        x = x.astype(np.float32)
    b = x.reshape(n, cols // 32, 32)
    kinds = rng.integers(0, 14, (n, cols // 32))
    for (i, j), kind in np.ndenumerate(kinds):
        if kind == 0:
            b[i, j] = 0
        elif kind == 1:
            b[i, j] = np.float32(2.0**-130) * rng.integers(-8, 9, 32)
        elif kind == 2:
            b[i, j, rng.integers(32)] = [np.nan, np.inf, -np.inf][rng.integers(3)]
        elif kind == 3:  # halves of code steps: ties
            b[i, j] = rng.integers(-24, 25, 32) * 0.25
        elif kind == 4:
            b[i, j] = rng.integers(-448, 449, 32)
        elif kind == 5:
            b[i, j] = np.float32(3e38) * rng.uniform(-1, 1, 32).astype(np.float32)
        elif kind == 6:
            b[i, j] = -0.0
        elif kind == 7:  # f32's smallest numbers beside 0
            b[i, j] = np.float32(1e-45) * rng.integers(-3, 4, 32)
    return mx.bf16(x) if bf16 else x


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,cols,gap", [(1, 32, 0), (1, 4096, 0), (7, 96, 0), (300, 160, 8), (33, 2048, 64), (5, 12320, 16),
                                        (1025, 64, 0)])
def test_quantize_and_back(dev, fmt, bf16, n, cols, gap):
    fmt = FMTS[fmt]
    say(f"quantize fmt {fmt} bf16 {bf16} n {n} cols {cols} gap {gap}")
    rng = np.random.default_rng(n * 7 + cols + fmt)
    x = rows_of_all_kinds(rng, n, cols, bf16)
    wide = np.full((n, cols + gap), np.float32(np.nan))
    wide[:, :cols] = x
    out = empty_rows(dev, n, cols, fmt)
    dtype = dr.DTYPE_BF16 if bf16 else dr.DTYPE_F32
    dr.mx_quantize(dev.ctx, put(dev, wide, bf16), n, cols, out, dtype=dtype, stride=cols + gap if gap else 0)
    codes, scales = get_rows(dev, out, n, cols)
    want_c, want_s = mx.quantise(x, fmt)
    assert np.array_equal(scales[:, : cols // 32], want_s[:, : cols // 32])
    assert np.array_equal(codes, want_c)
    # read back, both types; values past f32's largest are infinities
    want = mx.values(want_c, want_s, fmt, cols)
    for back in (False, True):
        dst = put(dev, np.full(n * cols + 64, 7.0), back)
        dr.mx_dequantize(dev.ctx, out, n, cols, dst, dtype=dr.DTYPE_BF16 if back else dr.DTYPE_F32)
        got = get(dev, dst, back)
        assert (got[n * cols:] == 7).all()
        with np.errstate(over="ignore"):
            w32 = want.astype(np.float32)
        w32 = mx.bf16(w32) if back else w32
        assert np.array_equal(got[: n * cols].reshape(n, cols), w32, equal_nan=True)


@pytest.mark.parametrize("fmt", list(FMTS))
def test_every_code_and_scale_reads_back(dev, fmt):
    fmt = FMTS[fmt]
    codes = np.arange(256, dtype=np.uint8)[None].repeat(256, 0)
    if fmt == dr.MX_E4M3:
        codes = codes.reshape(256, 256)
        scales = np.arange(256, dtype=np.uint8)[:, None].repeat(8, 1)
        cols = 256
    else:
        scales = np.arange(256, dtype=np.uint8)[:, None].repeat(16, 1)
        cols = 512
    out = dev.put(np.zeros(256 * cols, np.float32))
    dr.mx_dequantize(dev.ctx, put_rows(dev, codes, scales, fmt), 256, cols, out)
    with np.errstate(over="ignore"):
        want = mx.values(codes, scales, fmt, cols).astype(np.float32)
    assert np.array_equal(dev.get(out).reshape(256, cols), want, equal_nan=True)


def norm_reference(x, res, w, eps, bf16):
    """(held sum f32, y f64)."""
    h = (x.astype(np.float64) + (0 if res is None else res.astype(np.float64))).astype(np.float32)
    h = mx.bf16(h) if bf16 else h
    d = h.astype(np.float64)
    return h, d / np.sqrt((d * d).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * (1 if w is None else w.astype(np.float64))


def norm_error(y, cols):
    return np.abs(y) * ((cols / 2048 + 2) * 8 + 20) * 2.0**-24


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,cols,how", [(1, 4096, "total"), (1, 32, "plain"), (5, 96, "in x"), (300, 2048, "in residual"),
                                        (17, 2080, "no total"), (9, 3584, "stride"), (3, 8160, "no gain"), (4, 16384, "total"),
                                        (2, 16416, "in x"), (3, 40960, "no total"), (2, 65536, "in residual")])
def test_norm(dev, fmt, bf16, n, cols, how):
    fmt = FMTS[fmt]
    say(f"norm fmt {fmt} bf16 {bf16} n {n} cols {cols} {how}")
    rng = np.random.default_rng(n + cols + fmt)
    hold = mx.bf16 if bf16 else (lambda v: v.astype(np.float32))
    x = hold(rng.standard_normal((n, cols)).astype(np.float32))
    res = None if how in ("plain", "stride") else hold((rng.standard_normal((n, cols)) * 3).astype(np.float32))
    w = None if how == "no gain" else rng.uniform(0.2, 4, cols).astype(np.float32)
    if n > 2:
        x[1], w_zero = 0, res is None or how != "no gain"
        if res is not None and w_zero:
            res[1] = 0  # a row of zeros
    eps, dtype = 1e-5, dr.DTYPE_BF16 if bf16 else dr.DTYPE_F32
    stride = cols + 64 if how == "stride" else 0
    wide = np.full((n, cols + (64 if stride else 0)), np.float32(np.nan))
    wide[:, :cols] = x
    dx = put(dev, wide, bf16)
    dres = None if res is None else put(dev, res, bf16)
    total = {"total": put(dev, np.full((n, cols), 5.0), bf16), "stride": put(dev, np.full((n, cols), 5.0), bf16), "in x": dx,
             "in residual": dres}.get(how)
    out = empty_rows(dev, n, cols, fmt)
    dr.rms_norm_mx(dev.ctx, dx, n, cols, out, w=None if w is None else dev.put(w), eps=eps, residual=dres, total=total,
                   dtype=dtype, stride=stride)
    h, y = norm_reference(x, res, w, eps, bf16)
    if total is not None:
        assert np.array_equal(get(dev, total, bf16).reshape(n, cols), h)
    codes, scales = get_rows(dev, out, n, cols)
    mx.check_codes(codes, scales, fmt, y, norm_error(y, cols))


def test_norm_of_rows_without_an_answer(dev):
    """NaN and infinities stay in their rows; squares past f32's largest give zeros."""
    n, cols = 6, 256
    x = np.random.default_rng(3).standard_normal((n, cols)).astype(np.float32)
    x[1, 7], x[3, 200], x[4, 9] = np.nan, np.inf, 1e30
    out = empty_rows(dev, n, cols, dr.MX_E4M3)
    dr.rms_norm_mx(dev.ctx, dev.put(x), n, cols, out, eps=1e-6)
    codes, scales = get_rows(dev, out, n, cols)
    v = mx.values(codes, scales, dr.MX_E4M3, cols)
    assert np.isnan(v[1]).all()
    assert np.isnan(v[3, 192:224]).all() and (v[3, :192] == 0).all() and (v[3, 224:] == 0).all()  # inf / inf, finite / inf
    assert (v[4] == 0).all()
    _, y = norm_reference(x[[0, 2, 5]], None, None, 1e-6, False)
    mx.check_codes(codes[[0, 2, 5]], scales[[0, 2, 5]], dr.MX_E4M3, y, norm_error(y, cols))
