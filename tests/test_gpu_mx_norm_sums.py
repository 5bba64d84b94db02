"""The sum of squares of dr_rms_norm_mx in 64 bits: whatever a row's length, its codes are
those of a value within 8 * 2^-24 |y| of the exact one.  Eight squares are added in f32,
(eight roundings, of which the root takes half: 4), their sums in 64 bits, and the factor, its
product with h and the gain's round once each: 7, and second orders.

In rows of +-c all partial sums are alike and so are their roundings: an f32 sum of 512
eights a thread is off by more than that, which the last test shows without a GPU.
Needs an MI355X, but for that one."""
from __future__ import annotations

import numpy as np
import pytest

import dr_attn as dr
import mx_reference as mx
from test_gpu_mx_rows import FMTS, empty_rows, get_rows, norm_reference, put
from test_gpu_parity import dev, say, torch  # noqa: F401

EPS = 1e-6


def alike(rng, n, cols, c):
    """Rows of +-c, a gain that spreads their values between codes."""
    x = np.where(rng.random((n, cols)) < 0.5, -c, c).astype(np.float32)
    return x, rng.uniform(0.3, 3, cols).astype(np.float32)


def error(y):
    return np.abs(y) * 8 * 2.0**-24


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("kind", ["alike", "normal", "one large"])
@pytest.mark.parametrize("n,cols", [(3, 32), (300, 2048), (9, 3584), (4, 16384), (2, 16416), (2, 65536), (1, 1 << 22)])
def test_norm_of_long_rows(dev, fmt, kind, n, cols):
    fmt = FMTS[fmt]
    say(f"norm fmt {fmt} n {n} cols {cols} {kind}")
    rng = np.random.default_rng(n + cols)
    x, w = alike(rng, n, cols, C)
    if kind != "alike":
        x = rng.standard_normal((n, cols)).astype(np.float32)
    if kind == "one large":
        x[:, 5] = 4096
    out = empty_rows(dev, n, cols, fmt)
    dr.rms_norm_mx(dev.ctx, put(dev, x), n, cols, out, w=dev.put(w), eps=EPS)
    _, y = norm_reference(x, None, w, EPS, False)
    mx.check_codes(*get_rows(dev, out, n, cols), fmt, y, error(y))


C = np.float32(1.2345)


def test_the_check_sees_an_f32_sum():
    """Codes made with a factor from f32 sums, 4096 values of a thread by eights, are refused; those from a 64 bit sum pass."""
    rng = np.random.default_rng(0)
    cols = 1 << 22
    x, w = alike(rng, 1, cols, C)
    eight = np.float32(0)
    for _ in range(8):
        eight = np.float32(np.float64(C) * np.float64(C) + np.float64(eight))
    total = np.float32(0)
    for _ in range(512):
        total = np.float32(total + eight)
    _, y = norm_reference(x, None, w, EPS, False)
    for ss, passes in ((np.float64(total) / 4096, False), (np.float64(eight) / 8, True)):
        factor = np.float32(1 / np.sqrt(ss + np.float64(np.float32(EPS))))
        codes, scales = mx.quantise(x * factor * w, dr.MX_E4M3)
        if passes:
            mx.check_codes(codes, scales, dr.MX_E4M3, y, error(y))
        else:
            with pytest.raises(AssertionError):
                mx.check_codes(codes, scales, dr.MX_E4M3, y, error(y))
