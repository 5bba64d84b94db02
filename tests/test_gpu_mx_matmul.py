"""dr_mx_matmul and dr_mx_gated against tests/mx_reference.py (64 bits, on the
values that the codes stand for).

Tolerance of a sum of K products p, beside the output's own rounding (half a
step: 2^-24 of the value in f32, 2^-8 in bf16): the products are exact and each
addition rounds, or truncates, once to f32: K 2^-23 sum |p| at worst; signs
differ, so 4 sqrt(K) 2^-23 sum |p| is held to (and the whole, in the 2-norm, to
2^-22 of the sums of |p|).  In bf16 and in codes the 8 bit MFMA may be used,
which drops what lies 2^18 below the largest product of its 128: K 2^-18 max |p|
more.  Needs an MI355X."""
from __future__ import annotations

import numpy as np
import pytest

import dr_attn as dr
import mx_reference as mx
from test_gpu_mx_rows import FILL, FMTS, empty_rows, get, get_rows, put, put_rows
from test_gpu_parity import dev, say, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def weights(rng, rows, cols):
    """E2M1 rows of unequal size."""
    return mx.quantise((rng.standard_normal((rows, cols)) * np.exp(0.5 * rng.standard_normal((rows, 1)))
                        / np.sqrt(cols)).astype(np.float32), dr.MX_E2M1)


def acts(rng, n, cols, fmt):
    """Rows with channels of unequal size."""
    return mx.quantise((rng.standard_normal((n, cols)) * np.exp(0.8 * rng.standard_normal(cols))).astype(np.float32), fmt)


def product(w, a, fmt, cols, exact_sums, dev=None):
    """(sums, sums of magnitudes, what each sum may be off by), f64 (large ones on the device)."""
    wv, av = mx.values(*w, dr.MX_E2M1, cols), mx.values(*a, fmt, cols)
    if dev is not None and wv.size * av.shape[0] > 1 << 28:
        t = dev.t
        x, y = t.from_numpy(av).cuda(), t.from_numpy(np.ascontiguousarray(wv.T)).cuda()
        s, p = (x @ y).cpu().numpy(), (x.abs() @ y.abs()).cpu().numpy()
    else:
        s, p = av @ wv.T, np.abs(av) @ np.abs(wv).T
    tol = 4 * np.sqrt(cols) * 2.0**-23 * p
    if not exact_sums:
        tol = tol + cols * 2.0**-18 * np.abs(av).max(-1)[:, None] * np.abs(wv).max(-1)[None]
    return s, p, tol


# Up to 4 and 16 rows (many columns; more rows of weights than 16 a CU), and tiles of 16 x 32, 32 x 32, 64 x 32, 64 x 64,
# 64 x 128, 256 x 128 and 256 x 256 (tests/test_mx_refusals.py checks that no kernel is left out).
SIZES = [(1, 1, 32), (1, 16, 512), (1, 257, 544), (3, 100, 1056), (2, 130, 8224), (4, 33, 1024), (5, 48, 96), (16, 64, 2048),
         (13, 4200, 320), (17, 33, 96), (40, 130, 4096), (70, 48, 1120), (129, 300, 640), (129, 1028, 544), (260, 520, 416),
         (120, 4028, 1120), (513, 272, 1152), (513, 1028, 544), (250, 4028, 2336), (777, 1028, 32), (513, 8200, 544), (513, 8200, 1312),
         (2060, 4100, 1184), (1030, 12290, 1216)]


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,rows,cols", SIZES)
def test_matmul(dev, fmt, bf16, n, rows, cols):
    fmt = FMTS[fmt]
    say(f"matmul fmt {fmt} bf16 {bf16} n {n} rows {rows} cols {cols}")
    rng = np.random.default_rng(n * 3 + rows + cols + fmt)
    w, a = weights(rng, rows, cols), acts(rng, n, cols, fmt)
    w[1][:, cols // 32:] = 255  # bytes between scale rows are no scales
    a[1][:, cols // 32:] = 255
    dtype = dr.DTYPE_BF16 if bf16 else dr.DTYPE_F32
    s, p, tol = product(w, a, fmt, cols, not bf16, dev)
    half = 2.0**-8 if bf16 else 2.0**-24
    res = rng.standard_normal((n, rows)).astype(np.float32)
    res = mx.bf16(res) if bf16 else res
    dw, da = put_rows(dev, *w, dr.MX_E2M1), put_rows(dev, *a, fmt)
    for how in ("none", "apart", "in place"):
        want = s + (0 if how == "none" else res)
        buf = np.full(n * rows + 64, 7.0, np.float32)
        if how == "in place":
            buf[: n * rows] = res.reshape(-1)
        out = put(dev, buf, bf16)
        dr.mx_matmul(dev.ctx, dw, rows, cols, da, n, out, dtype=dtype,
                     residual={"none": None, "apart": put(dev, res, bf16), "in place": out}[how])
        got = get(dev, out, bf16)
        assert (got[n * rows:] == 7).all()
        err = np.abs(got[: n * rows].reshape(n, rows) - want)
        may = tol + half * (np.abs(want) + tol) * (1 if bf16 else 2)  # (f32: the sum and the addition round)
        say(f"  {how}: max err / bound {float((err / may).max()):.3g}")
        assert (err <= may).all()
        if not bf16 and how == "none":
            assert np.linalg.norm(err) <= 2.0**-22 * np.linalg.norm(p)
    # the bound sees one block of 32 columns missing
    cut = (a[0].copy(), a[1].copy())
    cut[0][:, -(16 if fmt == dr.MX_E2M1 else 32):] = 0
    assert (np.abs(product(w, cut, fmt, cols, True, dev)[0] - s) > tol).any()


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("to", list(FMTS))
@pytest.mark.parametrize("fn", [dr.ACT_SILU, dr.ACT_GELU], ids=["silu", "gelu"])
@pytest.mark.parametrize("n,rows,cols", [(1, 32, 32), (1, 160, 4096), (2, 288, 2080), (5, 96, 544), (12, 288, 2080), (16, 64, 96),
                                         (33, 288, 1056), (150, 352, 640), (300, 96, 2048), (520, 544, 160)])
def test_gated(dev, fmt, to, fn, n, rows, cols):
    fmt, to = FMTS[fmt], FMTS[to]
    say(f"gated fmt {fmt} to {to} fn {fn} n {n} rows {rows} cols {cols}")
    rng = np.random.default_rng(n + rows + cols + fmt)
    gate, up, a = weights(rng, rows, cols), weights(rng, rows, cols), acts(rng, n, cols, fmt)
    out = empty_rows(dev, n, rows, to)
    dr.mx_gated(dev.ctx, put_rows(dev, *gate, dr.MX_E2M1), put_rows(dev, *up, dr.MX_E2M1), rows, cols, put_rows(dev, *a, fmt), n,
                out, activation=fn)
    codes, scales = get_rows(dev, out, n, rows)
    check_gated(gate, up, a, fmt, cols, fn, codes, scales, to)


# tiles of 64 x 64 and 64 x 128, one and two a CU, 256 x 128 and 256 x 256
LARGE_GATED = [(100, 6176, 1184), (50, 18976, 544), (129, 6176, 1184), (129, 12320, 544), (513, 4128, 1056), (1030, 6176, 2080)]


@pytest.mark.parametrize("fmt,to,fn", [("e4m3", "e4m3", dr.ACT_SILU), ("e2m1", "e2m1", dr.ACT_GELU)], ids=["8bit", "4bit"])
@pytest.mark.parametrize("n,rows,cols", LARGE_GATED)
def test_gated_large(dev, fmt, to, fn, n, rows, cols):
    fmt, to = FMTS[fmt], FMTS[to]
    say(f"gated fmt {fmt} to {to} fn {fn} n {n} rows {rows} cols {cols}")
    rng = np.random.default_rng(n + rows + cols)
    gate, up, a = weights(rng, rows, cols), weights(rng, rows, cols), acts(rng, n, cols, fmt)
    out = empty_rows(dev, n, rows, to)
    dr.mx_gated(dev.ctx, put_rows(dev, *gate, dr.MX_E2M1), put_rows(dev, *up, dr.MX_E2M1), rows, cols, put_rows(dev, *a, fmt), n,
                out, activation=fn)
    codes, scales = get_rows(dev, out, n, rows)
    check_gated(gate, up, a, fmt, cols, fn, codes, scales, to, dev)


def check_gated(gate, up, a, fmt, cols, fn, codes, scales, to, dev=None):
    g, _, dg = product(gate, a, fmt, cols, False, dev)
    u, _, du = product(up, a, fmt, cols, False, dev)
    f = mx.act(g, fn)
    # |f'| <= 1.13 for both; f itself: e^z of |z| <= 100 or so to (|z| + 4) 2^-24, four more roundings; the product one
    df = 1.13 * dg + np.abs(f) * (np.abs(2 * g) + 2 * np.abs(g) ** 3 * 0.08 + 10) * 2.0**-24
    dy = df * np.abs(u) + np.abs(f) * du + df * du + np.abs(f * u) * 2.0**-24
    mx.check_codes(codes, scales, to, f * u, dy)


def test_scales_of_any_size(dev):
    """Powers of two from byte 0 to 254 on either side, as long as the values
    themselves are normal numbers."""
    rng = np.random.default_rng(5)
    n, rows, cols = 24, 32, 512
    for shift in (-100, -60, 0, 60, 100):
        w, a = weights(rng, rows, cols), acts(rng, n, cols, dr.MX_E4M3)
        w[1][:] = np.clip(w[1].astype(int) + shift, 0, 254)
        a[1][:] = np.clip(a[1].astype(int) - shift, 0, 254)
        for dtype in (dr.DTYPE_F32, dr.DTYPE_BF16):
            bf16 = dtype == dr.DTYPE_BF16
            s, _, tol = product(w, a, dr.MX_E4M3, cols, not bf16)
            out = put(dev, np.zeros(n * rows, np.float32), bf16)
            dr.mx_matmul(dev.ctx, put_rows(dev, *w, dr.MX_E2M1), rows, cols, put_rows(dev, *a, dr.MX_E4M3), n, out, dtype=dtype)
            got = get(dev, out, bf16).reshape(n, rows)
            assert (np.abs(got - s) <= tol + (2.0**-8 if bf16 else 2.0**-24) * (np.abs(s) + tol)).all(), shift


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 20, 300])
def test_nan_blocks(dev, fmt, bf16, n):
    """A block that stands for NaN makes NaN of its row's outputs and of no others,
    whatever it meets."""
    fmt = FMTS[fmt]
    rng = np.random.default_rng(n)
    rows, cols = 48, 672
    w, a = weights(rng, rows, cols), acts(rng, n, cols, fmt)
    w[1][5, 20] = a[1][n - 1, 3] = 255
    w[0][5, 20 * 16:21 * 16] = 0
    if n > 1:
        a[0][0] = 0  # NaN times 0 too
    out = put(dev, np.zeros(n * rows, np.float32), bf16)
    dr.mx_matmul(dev.ctx, put_rows(dev, *w, dr.MX_E2M1), rows, cols, put_rows(dev, *a, fmt), n, out,
                 dtype=dr.DTYPE_BF16 if bf16 else dr.DTYPE_F32)
    nan = np.zeros((n, rows), bool)
    nan[:, 5] = nan[n - 1] = True
    assert np.array_equal(np.isnan(get(dev, out, bf16).reshape(n, rows)), nan)
    hidden = empty_rows(dev, n, 64, dr.MX_E4M3)
    w2 = weights(rng, 64, cols)
    up = weights(rng, 64, cols)
    up[1][40, 0] = 255
    dr.mx_gated(dev.ctx, put_rows(dev, *w2, dr.MX_E2M1), put_rows(dev, *up, dr.MX_E2M1), 64, cols, put_rows(dev, *a, fmt), n, hidden)
    _, s = get_rows(dev, hidden, n, 64)
    want = np.zeros((n, 2), bool)
    want[:, 1] = want[n - 1] = True
    assert np.array_equal(s[:, :2] == 255, want)
