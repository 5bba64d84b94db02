"""Microscaled rows: what is refused before any device is touched, and the
format's reference itself (CPU only)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import dr_attn as dr
import mx_reference as mx

P = 4096  # an address that is aligned, never read: every call here is refused or empty


def rows(codes=P, scales=P, fmt=dr.MX_E4M3):
    return dr.CMxRows(codes, scales, fmt)


def refused(rc, *words, code=dr.DR_ERR_INVALID):
    assert rc == code, (rc, dr.load().dr_last_error())
    for w in words:
        assert w in dr.load().dr_last_error().decode()


def ctx():
    """A context's worth of zero bytes: device 0, no stream.  Refusals come before its use."""
    return ctypes.create_string_buffer(4096)


def test_null_context():
    lib, r = dr.load(), rows()
    refused(lib.dr_mx_quantize(None, P, 0, 1, 32, 0, r), "ctx")
    refused(lib.dr_mx_dequantize(None, r, 1, 32, P, 0), "ctx")
    refused(lib.dr_rms_norm_mx(None, P, None, None, 0, 1, 32, 0, None, 1e-6, r), "ctx")
    refused(lib.dr_mx_matmul(None, r, 1, 32, r, 1, P, None, 0), "ctx")
    refused(lib.dr_mx_gated(None, r, r, 32, 32, r, 1, 0, r), "ctx")


@pytest.mark.parametrize("cols", [0, 1, 31, 33, 48, (1 << 22) + 32])
def test_columns(cols):
    lib, c, r, w = dr.load(), ctx(), rows(), rows(fmt=dr.MX_E2M1)
    refused(lib.dr_mx_quantize(c, P, 0, 1, cols, 0, r), "cols", "32")
    refused(lib.dr_mx_dequantize(c, r, 1, cols, P, 0), "cols")
    refused(lib.dr_rms_norm_mx(c, P, None, None, 0, 1, cols, 0, None, 1e-6, r), "cols")
    refused(lib.dr_mx_matmul(c, w, 1, cols, r, 1, P, None, 0), "cols")
    refused(lib.dr_mx_gated(c, w, w, 32, cols, r, 1, 0, r), "cols")
    if cols:  # (0 rows: nothing to do)
        refused(lib.dr_mx_gated(c, w, w, cols, 32, r, 1, 0, r), "rows")


@pytest.mark.parametrize("bad,word", [(rows(codes=0), "NULL"), (rows(scales=0), "NULL"), (rows(codes=P + 8), "aligned"),
                                      (rows(scales=P + 2), "aligned"), (rows(fmt=2), "format"), (rows(fmt=-1), "format"),
                                      (None, "NULL")])
def test_rows(bad, word):
    lib, c, r, w = dr.load(), ctx(), rows(), rows(fmt=dr.MX_E2M1)
    refused(lib.dr_mx_quantize(c, P, 0, 1, 32, 0, bad), "out", word)
    refused(lib.dr_mx_dequantize(c, bad, 1, 32, P, 0), "rows", word)
    refused(lib.dr_rms_norm_mx(c, P, None, None, 0, 1, 32, 0, None, 1e-6, bad), "out", word)
    refused(lib.dr_mx_matmul(c, bad, 1, 32, r, 1, P, None, 0), "weights", word)
    refused(lib.dr_mx_matmul(c, w, 1, 32, bad, 1, P, None, 0), "act", word)
    refused(lib.dr_mx_gated(c, bad, w, 32, 32, r, 1, 0, r), "weights", word)
    refused(lib.dr_mx_gated(c, w, bad, 32, 32, r, 1, 0, r), "up", word)
    refused(lib.dr_mx_gated(c, w, w, 32, 32, bad, 1, 0, r), "act", word)
    refused(lib.dr_mx_gated(c, w, w, 32, 32, r, 1, 0, bad), "out", word)


def test_types_and_pointers():
    lib, c, r, w = dr.load(), ctx(), rows(), rows(fmt=dr.MX_E2M1)
    for bad in (-1, 2):
        refused(lib.dr_mx_quantize(c, P, bad, 1, 32, 0, r), "dtype")
        refused(lib.dr_mx_dequantize(c, r, 1, 32, P, bad), "dtype")
        refused(lib.dr_rms_norm_mx(c, P, None, None, bad, 1, 32, 0, None, 1e-6, r), "dtype")
        refused(lib.dr_mx_matmul(c, w, 1, 32, r, 1, P, None, bad), "dtype")
        refused(lib.dr_mx_gated(c, w, w, 32, 32, r, 1, bad, r), "activation")
    refused(lib.dr_mx_quantize(c, None, 0, 1, 32, 0, r), "x is NULL")
    refused(lib.dr_rms_norm_mx(c, None, None, None, 0, 1, 32, 0, None, 1e-6, r), "x is NULL")
    refused(lib.dr_mx_dequantize(c, r, 1, 32, None, 0), "out is NULL")
    refused(lib.dr_mx_dequantize(c, r, 1, 32, P + 4, 0), "aligned")
    refused(lib.dr_mx_matmul(c, w, 1, 32, r, 1, None, None, 0), "out is NULL")
    refused(lib.dr_mx_matmul(c, w, 1, 32, r, 1, P + 2, None, 0), "aligned")
    refused(lib.dr_mx_matmul(c, w, 1, 32, r, 1, P, P + 1, 1), "aligned")
    for args in ((P + 4, None, None, None), (P, P + 4, None, None), (P, None, P + 4, None), (P, None, None, P + 4)):
        x, res, total, gain = args
        refused(lib.dr_rms_norm_mx(c, x, res, total, 0, 1, 32, 0, gain, 1e-6, r), "aligned")
    # strides: shorter than a row, rows off 16 bytes, a sum over strided rows
    refused(lib.dr_mx_quantize(c, P, 0, 1, 64, 32, r), "overlap")
    refused(lib.dr_mx_quantize(c, P, 0, 1, 32, 34, r), "aligned")
    refused(lib.dr_mx_quantize(c, P, 1, 1, 32, 36, r), "aligned")
    refused(lib.dr_rms_norm_mx(c, P, None, P, 0, 2, 32, 64, None, 1e-6, r), "sum is x")
    # weights are 4 bit
    refused(lib.dr_mx_matmul(c, r, 1, 32, r, 1, P, None, 0), "not built", code=dr.DR_ERR_UNSUPPORTED)
    refused(lib.dr_mx_gated(c, r, w, 32, 32, r, 1, 0, r), "not built", code=dr.DR_ERR_UNSUPPORTED)
    refused(lib.dr_mx_gated(c, w, r, 32, 32, r, 1, 0, r), "not built", code=dr.DR_ERR_UNSUPPORTED)


def test_too_large():
    lib, c, r, w = dr.load(), ctx(), rows(), rows(fmt=dr.MX_E2M1)
    big = 1 << 40
    refused(lib.dr_mx_quantize(c, P, 0, big, 32, 0, r), "too large")
    refused(lib.dr_mx_dequantize(c, r, big, 32, P, 0), "too large")
    refused(lib.dr_rms_norm_mx(c, P, None, None, 0, big, 32, 0, None, 1e-6, r), "too large")
    refused(lib.dr_mx_matmul(c, w, big, 32, r, 1, P, None, 0), "too large")
    refused(lib.dr_mx_matmul(c, w, 1, 32, r, big, P, None, 0), "too large")
    refused(lib.dr_mx_gated(c, w, w, 32, 32, r, big, 0, r), "too large")


def test_nothing_to_do():
    lib, c, r, w = dr.load(), ctx(), rows(), rows(fmt=dr.MX_E2M1)
    assert lib.dr_mx_quantize(c, None, 0, 0, 32, 0, None) == dr.DR_OK
    assert lib.dr_mx_dequantize(c, None, 0, 32, None, 0) == dr.DR_OK
    assert lib.dr_rms_norm_mx(c, None, None, None, 0, 0, 32, 0, None, 1e-6, None) == dr.DR_OK
    assert lib.dr_mx_matmul(c, None, 0, 32, None, 5, None, None, 0) == dr.DR_OK
    assert lib.dr_mx_matmul(c, None, 5, 32, None, 0, None, None, 0) == dr.DR_OK
    assert lib.dr_mx_gated(c, None, None, 0, 32, None, 5, 0, None) == dr.DR_OK
    assert lib.dr_mx_gated(c, None, None, 32, 32, None, 0, 0, None) == dr.DR_OK


@pytest.mark.parametrize("fmt", [dr.MX_E2M1, dr.MX_E4M3])
def test_reference_codes(fmt):
    """code_values against the nearest of all codes, ties to the even one."""
    codes = mx.E2M1 if fmt == dr.MX_E2M1 else mx.e4m3_values()[:127]
    mid = (codes[1:] + codes[:-1]) / 2
    even = np.where(np.arange(len(mid)) % 2 == 0, codes[:-1], codes[1:])
    assert np.array_equal(mx.code_values(codes, fmt), codes)
    assert np.array_equal(mx.code_values(mid, fmt), even)
    y = np.random.default_rng(0).uniform(-codes[-1], codes[-1], 4000)
    y = np.concatenate([y, y / 16, y / 300])
    both = np.concatenate([codes, -codes])
    assert np.allclose(np.abs(mx.code_values(y, fmt) - y), np.abs(both[None] - y[:, None]).min(1), rtol=0, atol=0)
    assert np.array_equal(mx.encode(np.concatenate([codes, -codes]), fmt),
                          np.concatenate([np.arange(len(codes)), np.arange(len(codes)) + (8 if fmt == dr.MX_E2M1 else 128)]))


@pytest.mark.parametrize("fmt", [dr.MX_E2M1, dr.MX_E4M3])
def test_reference_scales(fmt):
    """The byte is the smallest that keeps the block within the largest code."""
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((300, 64)) * np.exp2(rng.integers(-60, 60, (300, 1)))).astype(np.float32)
    most = mx.TOP[fmt][0]
    x[0, :32], x[0, 32:] = 0, most  # nothing; exactly the largest code
    x[1, 0], x[1, 40] = np.nan, -np.inf
    x[2, 32:] = np.float32(2.0**-140)
    s = mx.scale_bytes(x, fmt).astype(int)
    a = np.abs(x.astype(np.float64)).reshape(300, 2, 32).max(-1)
    assert s[0].tolist() == [1, 127] and s[1].tolist() == [255, 255] and s[2, 1] == 1
    fine = np.isfinite(a)
    unit = np.exp2(s - 127.0)
    assert (a[fine] <= most * unit[fine]).all()
    assert ((a[fine] > most * unit[fine] / 2) | (s[fine] == 1)).all()
    c, sc = mx.quantise(x, fmt)
    v = mx.values(c, sc, fmt, 64)
    assert np.isnan(v[1]).all() and not np.isnan(np.delete(v, 1, 0)).any()


def test_plan():
    """Every kernel of the products is met by the sizes of tests/test_gpu_mx_matmul.py, and
    by the 256 compute units that those are for; the plan's own refusals."""
    from test_gpu_mx_matmul import LARGE_GATED, SIZES

    met = {dr.mx_plan(rows, cols, n, act_format=f, dtype=d) for n, rows, cols in SIZES for f in (0, 1) for d in (0, 1)}
    assert met == set(range(10))
    assert [dr.mx_plan(rows, cols, n, gated=True) for n, rows, cols in LARGE_GATED] == [6, 6, 7, 7, 8, 9]
    assert {dr.mx_plan(64, 512, n, gated=True) for n in (1, 4, 5, 16, 17, 100)} == {0, 1, 3}
    # f32 sums of 8 bit codes never take the block-scaled MFMA's kernels, others never the bf16 MFMA's tile
    for n in (1, 16, 17, 100, 1000, 10000):
        assert dr.mx_plan(4096, 4096, n) <= 5
        assert 5 not in (dr.mx_plan(4096, 4096, n, act_format=dr.MX_E2M1), dr.mx_plan(4096, 4096, n, dtype=dr.DTYPE_BF16))
    for bad in (dict(rows=0, cols=32, n=1), dict(rows=1, cols=31, n=1), dict(rows=1, cols=32, n=0), dict(rows=1, cols=32, n=1, n_cu=0),
                dict(rows=1, cols=32, n=1, dtype=3), dict(rows=1 << 40, cols=32, n=1)):
        with pytest.raises(dr.DrError):
            dr.mx_plan(**bad)


@pytest.mark.parametrize("gated", [False, True], ids=["product", "gated"])
@pytest.mark.parametrize("dtype", [dr.DTYPE_F32, dr.DTYPE_BF16], ids=["f32", "bf16"])
def test_grids(gated, dtype):
    """The largest sizes that are taken launch fewer than 2^32 lanes."""
    tile = {2: (16, 32), 3: (32, 32), 4: (64, 32), 5: (64, 64), 6: (64, 64), 7: (64, 128), 8: (128 if gated else 256, 128),
            9: (128 if gated else 256, 256)}
    most = (2**31 - 1) // 256
    for n in [1, 4, 5, 16, 17, 31, 32, 33, 64, 65, 127, 129, 1000, 2047, 2048, 2049, 2080, 2081, 4000, 2**16, 2**20 + 1, most]:
        rows = min(most, 2**34 // n)
        for rows in {rows, rows - 31, rows // 2 + 1}:
            rows = rows // 32 * 32 if gated else rows
            kernel = dr.mx_plan(rows, 4096, n, gated=gated, dtype=dtype)
            columns, acts = tile.get(kernel, (32 if gated else 16, n))
            lanes = -(-rows // columns) * -(-n // acts) * (512 if kernel != 0 or not gated else 256)  # (or fewer)
            assert lanes < 2**32, (n, rows, kernel)
