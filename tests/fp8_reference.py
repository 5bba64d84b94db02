"""The DR_PRECISION_FP8 cache format and the attention over it in float64, written
from their definitions (include/dr_attn.h), for the tests."""
from __future__ import annotations

import math

import numpy as np


def e4m3_round(y: np.ndarray) -> np.ndarray:
    """float64 -> nearest e4m3 value (ties to even); |y| <= 448."""
    mag = np.maximum(np.abs(y), 2.0 ** -6)  # smallest normal: the step below is that of 2^-6
    _, e = np.frexp(mag)
    step = np.ldexp(1.0, e - 4)
    return np.rint(y / step) * step


def stored(x: np.ndarray) -> np.ndarray:
    """The values that f32 rows [..., head_dim] stand for once stored."""
    x = np.asarray(x, np.float32).astype(np.float64)
    bad = ~np.isfinite(x).all(-1, keepdims=True)
    x = np.where(bad, 0.0, x)
    top = np.abs(x).max(-1, keepdims=True)
    m, e = np.frexp(top)
    e = np.maximum(e - 9 + (m > 0.875), -126)
    y = np.ldexp(e4m3_round(np.ldexp(x, -e)), e)
    return np.where(bad, np.nan, y)


def attend(q, k, v, pos, scale, window=None, prefix=None):
    """(out, weighted) of one batch slot: q [n, heads, hd] at positions pos,
    k and v [keys, kv heads, hd] (a NaN counts only where it is visible).  out
    [n, heads, hd] in float64; weighted: the same sums over |v|."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    n, heads, hd = q.shape
    keys, hkv, _ = k.shape
    qp, kp = np.asarray(pos, np.int64)[:, None], np.arange(keys)[None, :]
    see = np.ones((n, keys), bool)
    if window is not None:
        see &= np.abs(qp - kp) < window
    if prefix is not None:
        see &= ~((qp < prefix) & (kp > qp))
    out, weighted = np.full((n, heads, hd), np.nan), np.full((n, heads, hd), np.nan)
    for h in range(heads):
        g = h // (heads // hkv)
        kn, vn = np.isnan(k[:, g]).any(-1), np.isnan(v[:, g]).any(-1)
        s = (q[:, h] @ np.nan_to_num(k[:, g]).T) * float(np.float32(scale))
        s = np.where(see, s, -np.inf)
        m = s.max(1, keepdims=True)
        p = np.where(see, np.exp(s - np.where(np.isfinite(m), m, 0.0)), 0.0)
        ok = see.any(1) & ~(see & (kn | vn)).any(1)
        l = np.where(ok, p.sum(1), 1.0)[:, None]
        out[ok, h] = ((p @ np.nan_to_num(v[:, g])) / l)[ok]
        weighted[ok, h] = ((p @ np.abs(np.nan_to_num(v[:, g]))) / l)[ok]
    return out, weighted


def bound(q, k, v, weighted, out, scale, bf16: bool) -> np.ndarray:
    """How far the kernel's outputs may be from attend()'s.  q is exact (f32, or
    bf16 rows), k and v are what the cache holds.

    Scores: q is held in two f16 planes (2^-22 of each value; bf16 exactly), the
    products are summed in f32 (hd terms and the planes: (hd + 4) 2^-24 of the sum
    of their sizes, twice for the two planes); s - m is rounded once and exp2
    takes 2 steps of 2^-23.  A score off by ds changes p by exp(ds) - 1, an output
    by at most twice that of the weighted |v|.  p is held to 2^-22 (bf16 rows: the
    half step of f16, 2^-11); sums over keys in f32 (keys 2^-24); the smallest p
    that f16 tells from 0 is 2^-25 of units in which the row's largest is at least
    2^8, times the largest value per key.  bf16 output: half a step, 2^-8."""
    hd, keys = q.shape[-1], k.shape[0]
    qa, ka = np.abs(np.asarray(q, np.float64)), np.nan_to_num(np.abs(k))
    heads, hkv = q.shape[1], k.shape[1]
    size = np.stack([(qa[:, h] @ ka[:, h // (heads // hkv)].T).max(1) for h in range(heads)], 1)[..., None]
    size = size * abs(scale)
    ds = size * (2.0 ** -22 + 2 * (hd + 4) * 2.0 ** -24) + (2 * size + 16) * 2.0 ** -23
    rel = 2 * np.expm1(ds) + (2.0 ** -11 if bf16 else 2.0 ** -22) + (keys + 8) * 2.0 ** -23
    vmax = np.nan_to_num(np.abs(v)).max() if v.size else 0.0
    tol = weighted * rel + keys * 2.0 ** -33 * vmax
    return tol + (np.abs(out) + tol) * 2.0 ** -8 if bf16 else tol


def check(got, want, tol, what=""):
    got = np.asarray(got, np.float64).reshape(want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN pattern differs"
    ok = ~np.isnan(want)
    if not ok.any():
        return 0.0
    over = np.abs(got - want)[ok] / np.maximum(tol[ok], 1e-300)
    worst = float(np.where(np.abs(got - want)[ok] == 0, 0.0, over).max())
    assert worst <= 1.0, f"{what}: {worst:.2f} of the bound, max-abs {np.abs(got - want)[ok].max():.3e}"
    return worst


def default_scale(hd: int) -> float:
    return 1.0 / math.sqrt(hd)
