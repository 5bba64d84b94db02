"""Microscaled rows and the operators on them in 64 bits, in numpy (include/dr_attn.h,
dr_mx_rows): written from the format's definition, without the library."""
from __future__ import annotations

import numpy as np

import dr_attn as dr

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
TOP = {dr.MX_E2M1: (6.0, 2), dr.MX_E4M3: (448.0, 8)}  # the largest code, its exponent
NAN = 255


def e4m3_values() -> np.ndarray:
    """The value of each of the 256 codes."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7), m / 8 * 2.0**-6)
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


def scale_bytes(x: np.ndarray, fmt: int) -> np.ndarray:
    """The scale byte of each block of rows x [n][cols]."""
    n, cols = x.shape
    a = np.abs(x.astype(np.float64)).reshape(n, cols // 32, 32).max(-1)
    most, top = TOP[fmt]
    _, e = np.frexp(np.where(np.isfinite(a) & (a > 0), a, 1.0))
    e = e - 1 - top
    e = np.maximum(np.where(a > most * np.exp2(e.astype(np.float64)), e + 1, e), -126)
    return np.where(np.isfinite(a), np.where(a > 0, e, -126) + 127, NAN).astype(np.uint8)


def code_values(y: np.ndarray, fmt: int) -> np.ndarray:
    """y (a value over its block's 2^e) rounded to the nearest code's value, ties to even."""
    bits, low, most = (1, 0, 6.0) if fmt == dr.MX_E2M1 else (3, -6, 448.0)
    mag = np.maximum(np.abs(y), 2.0**low)
    _, g = np.frexp(mag)
    step = np.exp2((g - 1 - bits).astype(np.float64))
    return np.clip(np.rint(y / step) * step, -most, most)


def encode(v: np.ndarray, fmt: int) -> np.ndarray:
    """Code numbers of exact code values (signed zeros kept)."""
    sign = np.signbit(v)
    if fmt == dr.MX_E2M1:
        return (np.searchsorted(E2M1, np.abs(v)) + 8 * sign).astype(np.uint8)
    pos = e4m3_values()[:127]
    return (np.searchsorted(pos, np.abs(v)) + 128 * sign).astype(np.uint8)


def quantise(x: np.ndarray, fmt: int):
    """(codes, scales) of rows x, laid out as dr_mx_rows; gap bytes 0."""
    n, cols = x.shape
    s = scale_bytes(x, fmt)
    bad = np.repeat(s == NAN, 32, axis=1)
    unit = np.exp2(np.repeat(s, 32, axis=1).astype(np.float64) - 127)
    y = np.where(bad, 0.0, x.astype(np.float64)) / np.where(bad, 1.0, unit)
    c = encode(code_values(y, fmt), fmt)
    c[bad] = 0
    if fmt == dr.MX_E2M1:
        c = c[:, 0::2] | c[:, 1::2] << 4
    scales = np.zeros((n, dr.mx_pitch(cols)), np.uint8)
    scales[:, : cols // 32] = s
    return np.ascontiguousarray(c), scales


def values(codes: np.ndarray, scales: np.ndarray, fmt: int, cols: int) -> np.ndarray:
    """The f64 values that rows stand for."""
    n = codes.shape[0]
    if fmt == dr.MX_E2M1:
        c = np.stack((codes & 15, codes >> 4), -1).reshape(n, cols)
        v = np.where(c & 8, -E2M1[c & 7], E2M1[c & 7])
    else:
        v = e4m3_values()[codes]
    s = np.repeat(scales[:, : cols // 32], 32, axis=1)
    return np.where(s == NAN, np.nan, v * np.exp2(s.astype(np.float64) - 127))


def bf16(x: np.ndarray) -> np.ndarray:
    """f32 values rounded to bf16 (nearest, ties to even), as f32."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    b = (b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000
    out = b.astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.float32(np.nan), out)


def act(x: np.ndarray, fn: int) -> np.ndarray:
    """The gated block's activation (f64)."""
    z = x if fn == dr.ACT_SILU else 2 * np.sqrt(2 / np.pi) * (x + 0.044715 * x**3)
    with np.errstate(over="ignore"):
        return x / (1 + np.exp(-z))


def check_codes(codes, scales, fmt: int, y: np.ndarray, dy: np.ndarray) -> None:
    """codes and scales are a quantisation of some y' with |y' - y| <= dy: a
    block's byte lies between those of its smallest and largest possible
    magnitude, each code between those of its smallest and largest possible value."""
    n, cols = y.shape
    blocks = lambda v: v.reshape(n, cols // 32, 32)  # noqa: E731
    s = scales[:, : cols // 32]
    lo = scale_bytes(blocks(np.maximum(np.abs(y) - dy, 0)).max(-1).repeat(32, axis=1).reshape(n, cols), fmt)
    hi = scale_bytes(blocks(np.abs(y) + dy).max(-1).repeat(32, axis=1).reshape(n, cols), fmt)
    assert ((s >= lo) & (s <= hi)).all(), "a scale byte"
    unit = np.exp2(np.repeat(s, 32, axis=1).astype(np.float64) - 127)
    got = values(codes, scales, fmt, cols) / unit
    down, up = code_values((y - dy) / unit, fmt), code_values((y + dy) / unit, fmt)
    bad = ~((got >= down) & (got <= up))
    assert not bad.any(), (int(bad.sum()), got[bad][:4], down[bad][:4], up[bad][:4])
