"""The sums of dr_mx_gated are f32 sums of exact products, whatever its size and types.

Products that cancel.  Of eight columns two hold the largest products, P and -P, and
one the smallest, all of them a code times a code: what is left is the smallest, an
exact number, so that f32 sums in any order are exact and the output is f(g) u to the
activation's own error, (|2 g| + 0.16 |g|^3 + 10) 2^-24, and one rounding.

Sums in general, beside check_gated's with the f32 bound (4 sqrt(K) 2^-23 of the sums of
magnitudes P), by how many codes differ: K / 8 additions that are each off by 2^-24 of a partial sum of P
/ sqrt(K), at random or (truncated) all one way by half of 2^-23, leave (1 + sqrt(K) / 16) 2^-24 P.
A value that may be off by dy meets a border between two codes with probability 2 dy /
step and is then off by a step: errors in steps have squares that add up to sum 2 dy / step, held to
4 times that and eight more.  Needs an MI355X, but for the last test."""
from __future__ import annotations

import numpy as np
import pytest

import dr_attn as dr
import mx_reference as mx
from test_gpu_mx_matmul import acts, product, weights
from test_gpu_mx_rows import FMTS, empty_rows, get_rows, put_rows
from test_gpu_parity import dev, say, torch  # noqa: F401

gpu = pytest.mark.gpu


def steps(y, fmt):
    """The distance between codes around each value of rows y."""
    unit = np.exp2(mx.scale_bytes(y, fmt).astype(np.float64) - 127).repeat(32, axis=1)
    bits, low = (1, 0) if fmt == dr.MX_E2M1 else (3, -6)
    _, e = np.frexp(np.maximum(np.abs(y) / unit, 2.0**low))
    return np.exp2((e - 1 - bits).astype(np.float64)) * unit


def check_sums(gate, up, a, fmt, cols, fn, codes, scales, to, dev=None):
    g, pg, dg = product(gate, a, fmt, cols, True, dev)
    u, pu, du = product(up, a, fmt, cols, True, dev)
    f = mx.act(g, fn)
    own = np.abs(f) * (np.abs(2 * g) + 2 * np.abs(g) ** 3 * 0.08 + 10) * 2.0**-24
    off = lambda x, v: (1.13 * x + own) * np.abs(u) + np.abs(f) * v + (1.13 * x + own) * v + np.abs(f * u) * 2.0**-24  # noqa: E731
    y = f * u
    mx.check_codes(codes, scales, to, y, off(dg, du))
    usual = (1 + np.sqrt(cols) / 16) * 2.0**-24
    step = steps(y, to)
    err = (mx.values(codes, scales, to, y.shape[1]) - mx.values(*mx.quantise(y, to), to, y.shape[1])) / step
    allowed = 4 * (2 * off(usual * pg, usual * pu) / step).sum() + 8
    say(f"  squares: {(err**2).sum():.4g}, {allowed:.4g} allowed")
    assert (err**2).sum() <= allowed


def run(dev, gate, up, a, rows, cols, n, fmt, to, fn):
    out = empty_rows(dev, n, rows, to)
    dr.mx_gated(dev.ctx, put_rows(dev, *gate, dr.MX_E2M1), put_rows(dev, *up, dr.MX_E2M1), rows, cols, put_rows(dev, *a, fmt), n,
                out, activation=fn)
    return get_rows(dev, out, n, rows)


# every kernel of the block: strips for 4 and 16 rows, tiles of 32 x 32, 64 x 64 (one and two a CU),
# 64 x 128 (the same), 256 x 128, 256 x 256
SIZES = [(3, 64, 544), (16, 96, 4096), (17, 64, 544), (33, 288, 1056), (100, 96, 4096), (50, 6176, 544), (100, 6176, 1184), (50, 18976, 544),
         (129, 6176, 1184), (129, 12320, 544), (513, 4128, 1056), (1030, 6176, 2080)]


@gpu
@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("n,rows,cols", SIZES)
def test_products_that_cancel(dev, fmt, n, rows, cols):
    fmt = FMTS[fmt]
    say(f"cancelling products fmt {fmt} n {n} rows {rows} cols {cols}")
    rng = np.random.default_rng(n + rows + cols)
    big, small = (448.0, 2.0**-6) if fmt == dr.MX_E4M3 else (6.0, 0.5)
    av, wv = np.zeros((n, cols)), np.zeros((rows, cols))
    at = rng.integers(0, cols // 8)
    av[:, 8 * at + 1] = av[:, 8 * at + 6] = big
    av[:, 8 * at + 3] = small * rng.integers(1, 4, n)
    wv[:, 8 * at + 1], wv[:, 8 * at + 6] = 6, -6
    wv[:, 8 * at + 3] = rng.choice([0.5, 1, -0.5, 1.5], rows)
    blocks = cols // 32
    lift = 4 if fmt == dr.MX_E4M3 else 0  # products of about 1 / 4

    def rows_of(v, f, byte):
        c = mx.encode(v, f)
        c = np.ascontiguousarray(c[:, 0::2] | c[:, 1::2] << 4) if f == dr.MX_E2M1 else c
        s = np.zeros((len(v), dr.mx_pitch(cols)), np.uint8)
        s[:, :blocks] = byte
        return c, s

    w, a = rows_of(wv, dr.MX_E2M1, 127 + lift), rows_of(av, fmt, 127)
    codes, scales = run(dev, w, w, a, rows, cols, n, fmt, dr.MX_E4M3, dr.ACT_SILU)
    g = mx.values(*a, fmt, cols) @ mx.values(*w, dr.MX_E2M1, cols).T
    assert np.array_equal(np.float32(g), g) and (g != 0).all()
    y = mx.act(g, dr.ACT_SILU) * g
    mx.check_codes(codes, scales, dr.MX_E4M3, y, np.abs(y) * (np.abs(2 * g) + 0.16 * np.abs(g) ** 3 + 11) * 2.0**-24)


@gpu
@pytest.mark.parametrize("fmt,to,fn", [("e4m3", "e4m3", dr.ACT_SILU), ("e4m3", "e2m1", dr.ACT_GELU), ("e2m1", "e4m3", dr.ACT_GELU)],
                         ids=["8bit", "8to4", "4to8"])
@pytest.mark.parametrize("n,rows,cols", SIZES)
def test_gated_sums(dev, fmt, to, fn, n, rows, cols):
    fmt, to = FMTS[fmt], FMTS[to]
    say(f"gated sums fmt {fmt} to {to} fn {fn} n {n} rows {rows} cols {cols}")
    rng = np.random.default_rng(n * 5 + rows + cols + fmt)
    gate, up, a = weights(rng, rows, cols), weights(rng, rows, cols), acts(rng, n, cols, fmt)
    check_sums(gate, up, a, fmt, cols, fn, *run(dev, gate, up, a, rows, cols, n, fmt, to, fn), to, dev)


@gpu
@pytest.mark.parametrize("n", [12, 40, 300])
def test_wide_channels(dev, n):
    """A few channels far larger than the rest, as behind a norm's gain: most codes of their blocks are small."""
    rng = np.random.default_rng(n)
    rows, cols = 256, 2048
    gain = np.exp(0.5 * rng.standard_normal(cols)) * np.where(rng.random(cols) < 0.01, 64, 1)
    gate, up = weights(rng, rows, cols), weights(rng, rows, cols)
    a = mx.quantise((rng.standard_normal((n, cols)) * gain).astype(np.float32), dr.MX_E4M3)
    check_sums(gate, up, a, dr.MX_E4M3, cols, dr.ACT_SILU, *run(dev, gate, up, a, rows, cols, n, dr.MX_E4M3, dr.MX_E4M3, dr.ACT_SILU),
               dr.MX_E4M3)


@pytest.mark.parametrize("noise", [0.0, 1e-3])
@pytest.mark.parametrize("n,rows,cols", [(3, 64, 544), (16, 96, 4096), (33, 288, 1056)])
def test_the_check_sees_noise(noise, n, rows, cols):
    """Sums that are off by 1e-3 of their usual size are refused, exact ones pass (no GPU)."""
    rng = np.random.default_rng(n)
    gate, up, a = weights(rng, rows, cols), weights(rng, rows, cols), acts(rng, n, cols, dr.MX_E4M3)
    g, u = (product(w, a, dr.MX_E4M3, cols, True)[0] for w in (gate, up))
    g, u = (v + noise * np.sqrt((v * v).mean()) * rng.standard_normal(v.shape) for v in (g, u))
    codes, scales = mx.quantise(mx.act(g, dr.ACT_SILU) * u, dr.MX_E4M3)
    if noise:
        with pytest.raises(AssertionError):
            check_sums(gate, up, a, dr.MX_E4M3, cols, dr.ACT_SILU, codes, scales, dr.MX_E4M3)
    else:
        check_sums(gate, up, a, dr.MX_E4M3, cols, dr.ACT_SILU, codes, scales, dr.MX_E4M3)
