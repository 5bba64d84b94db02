"""Blocks of very unequal scales within the 128 columns of a step.

Where f32 sums of exact products are promised: few products, all multiples of one
unit and of a sum of magnitudes below 2^24 units, so that f32 sums are exact in any order:
the outputs equal the exact ones, with the largest product 2^21 to 2^23 times the smallest and
large ones that cancel, in the same eight columns, in the same block and over blocks.

Elsewhere (8 bit activations to bf16, more than 16 rows): random codes of every size, off by 2^-10 of
the sum of magnitudes at most (seven of eight products lose less than 2^-13 of the largest each, the
f32 sums sqrt(K) 2^-23 of it), beside bf16's own rounding.  Needs an MI355X."""
from __future__ import annotations

import numpy as np
import pytest

import dr_attn as dr
import mx_reference as mx
from test_gpu_mx_matmul import acts, weights
from test_gpu_mx_rows import FMTS, get, put, put_rows
from test_gpu_parity import dev, say, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def rows_of(v, fmt, scales):
    """Codes of the code values v with the given scale bytes."""
    c = mx.encode(v, fmt)
    c = np.ascontiguousarray(c[:, 0::2] | c[:, 1::2] << 4) if fmt == dr.MX_E2M1 else c
    s = np.zeros((len(v), dr.mx_pitch(v.shape[1])), np.uint8)
    s[:, : v.shape[1] // 32] = scales
    return c, s


@pytest.mark.parametrize("fmt,bf16", [("e2m1", False), ("e2m1", True), ("e4m3", False)], ids=["4bit", "4bit-bf16", "8bit"])
@pytest.mark.parametrize("n,rows,cols", [(1, 40, 128), (4, 40, 544), (16, 300, 1056), (17, 33, 128), (40, 130, 544), (300, 96, 1056),
                                         (520, 520, 544), (513, 8200, 160), (2060, 4100, 160)])
def test_far_scales(dev, fmt, bf16, n, rows, cols):
    fmt = FMTS[fmt]
    say(f"far scales fmt {fmt} bf16 {bf16} n {n} rows {rows} cols {cols}")
    rng = np.random.default_rng(n + rows + cols)
    blocks = cols // 32
    for far in (12, 14):  # the products of one block of four are 2^far times the others'
        ws, as_ = np.full(blocks, 127), np.full(blocks, 127)
        large = rng.integers(0, min(4, blocks)) + 4 * rng.integers(0, max(blocks // 4, 1))
        ws[large], as_[large] = 127 + far // 2, 127 + far - far // 2
        wv, av = np.zeros((rows, cols)), np.zeros((n, cols))
        at = np.concatenate([b * 32 + rng.permutation(32)[:4] for b in range(min(blocks, 8)) if b != large])  # (28 at most)
        wv[:, at] = rng.choice([0.5, -0.5, 1, -1.5, 3], (rows, len(at)))
        av[:, at] = rng.choice([0.5, -0.5, 1, 1.5, -2], (n, len(at)))
        first = large * 32 + 8 * rng.integers(0, 4)  # +P and -P within eight columns; 1.5 P and -1.5 P over two eights
        other = large * 32 + 8 * ((first // 8 + 1) % 4)
        for p, q, v in ((first + 1, first + 6, 6.0), (first + 3, other + 2, 3.0)):
            wv[:, p], wv[:, q] = v, -v
            av[:, p] = av[:, q] = 6
        w, a = rows_of(wv, dr.MX_E2M1, ws), rows_of(av, fmt, as_)
        x, y = mx.values(*a, fmt, cols), mx.values(*w, dr.MX_E2M1, cols)
        s, p = x @ y.T, np.abs(x) @ np.abs(y).T
        assert p.max() < 2.0**24 * 0.25 and (s != 0).any()
        out = put(dev, np.zeros(n * rows, np.float32), bf16)
        dr.mx_matmul(dev.ctx, put_rows(dev, *w, dr.MX_E2M1), rows, cols, put_rows(dev, *a, fmt), n, out,
                     dtype=dr.DTYPE_BF16 if bf16 else dr.DTYPE_F32)
        want = s.astype(np.float32)
        assert np.array_equal(get(dev, out, bf16).reshape(n, rows), mx.bf16(want) if bf16 else want)


@pytest.mark.parametrize("n,rows,cols", [(17, 33, 128), (40, 130, 4096), (129, 1028, 544), (300, 96, 1056), (520, 520, 544), (513, 8200, 544),
                                         (2060, 4100, 544)])
def test_what_bf16_outputs_lose(dev, n, rows, cols):
    say(f"8 bit codes of every size n {n} rows {rows} cols {cols}")
    rng = np.random.default_rng(n)
    a = acts(rng, n, cols, dr.MX_E4M3)
    c = rng.integers(0, 256, (n, cols), dtype=np.uint8)
    a = (np.where((c & 127) == 127, 0, c).astype(np.uint8), a[1])
    w = weights(rng, rows, cols)
    a[1][:, : cols // 32] += rng.integers(0, 12, (n, cols // 32)).astype(np.uint8)
    x, y = mx.values(*a, dr.MX_E4M3, cols), mx.values(*w, dr.MX_E2M1, cols)
    s, p = x @ y.T, np.abs(x) @ np.abs(y).T
    out = put(dev, np.zeros(n * rows, np.float32), True)
    dr.mx_matmul(dev.ctx, put_rows(dev, *w, dr.MX_E2M1), rows, cols, put_rows(dev, *a, dr.MX_E4M3), n, out, dtype=dr.DTYPE_BF16)
    tol = (2.0**-10 + np.sqrt(cols) * 2.0**-23) * p
    err = np.abs(get(dev, out, True).reshape(n, rows) - s)
    beyond = np.maximum(err - 2.0**-8 * (np.abs(s) + tol), 0)
    say(f"  largest error beside the rounding {float((beyond / p).max()):.3g} of the sum of magnitudes")
    assert (beyond <= tol).all()


@pytest.mark.parametrize("fmt", list(FMTS))
@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 16, 20, 300])
def test_ends_of_the_scales(dev, fmt, bf16, n):
    """Largest codes at the largest scale whose values are f32 numbers, and values down to 2^-126, times weights of the other end."""
    fmt = FMTS[fmt]
    rng = np.random.default_rng(n)
    rows, cols = 48, 160
    top, most, low = (246, 448.0, 10) if fmt == dr.MX_E4M3 else (252, 6.0, 2)  # (smallest codes 2^-9 and 2^-1)
    for byte, weight_byte in ((top, 20), (low, 220)):
        av = np.where(rng.random((n, cols)) < 0.5, most, 1.0) * rng.choice([1, -1], (n, cols))
        if byte == low:
            av[:, ::7] = 2.0**-9 if fmt == dr.MX_E4M3 else 0.5
        wv = rng.choice([0.5, 1, -1.5, 2, -3, 6, 0], (rows, cols))
        a, w = rows_of(av, fmt, byte), rows_of(wv, dr.MX_E2M1, weight_byte)
        x, y = mx.values(*a, fmt, cols), mx.values(*w, dr.MX_E2M1, cols)
        s, p = x @ y.T, np.abs(x) @ np.abs(y).T
        out = put(dev, np.zeros(n * rows, np.float32), bf16)
        dr.mx_matmul(dev.ctx, put_rows(dev, *w, dr.MX_E2M1), rows, cols, put_rows(dev, *a, fmt), n, out,
                     dtype=dr.DTYPE_BF16 if bf16 else dr.DTYPE_F32)
        lossy = bf16 and fmt == dr.MX_E4M3 and n > 16
        tol = (4 * np.sqrt(cols) * 2.0**-23 + (2.0**-10 if lossy else 0)) * p
        err = np.abs(get(dev, out, bf16).reshape(n, rows) - s)
        assert (err <= tol + (2.0**-8 if bf16 else 2.0**-24) * (np.abs(s) + tol)).all(), byte
