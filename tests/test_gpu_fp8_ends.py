"""Attention over DR_PRECISION_FP8 layers at the ends of what f32 holds: rows so
small that their scale is the smallest, sizes that grow from tile to tile, query
rows near f32's smallest numbers, rows out of sight that are larger than those
in sight by less than what takes the slow way, a scale that is no number.  Needs
an MI355X."""
from __future__ import annotations

import math

import numpy as np
import pytest

import dr_attn as dr
from fp8_reference import attend, bound, check, stored
from helpers import bf16_round

from test_gpu_fp8_attention import Problem, empty_rows, put_rows, rows_of
from test_gpu_fp8_far_scales import BF16, SHAPES, visible
from test_gpu_fp8_wide import wave_rows
from test_gpu_parity import dev, say, torch  # noqa: F401

pytestmark = pytest.mark.gpu

SMALL = pytest.mark.parametrize("size", [1.2e-36, 1e-40])  # (most rows' largest values below 1.75 * 2^-118: the smallest scale)



def run(dev, p, wave, bf16, window=None, prefix=None, split=0, scale=None, more=None):
    """A call checked row by row against the bound of the keys that it sees (as
    for scales far apart), `more(i, seen keys)` added to it, and a floor for rows
    near f32's smallest numbers: up to 8 waves' parts and their sums in up to 3
    splits, and the splits' sum, are each rounded to 2^-150 at worst, less than
    64 roundings of a row whose weights add up to 2^-8 or more: 2^-136.  (bf16's
    subnormals are 2^-126 / 2^7 = 2^-133 apart, so a row of them is off by half of
    that where the relative 2^-8 says less.)"""
    scale = 1 / math.sqrt(p.hd) if scale is None else scale
    if bf16:
        p.q = bf16_round(p.q)
    cache = dr.StepCache(dev.ctx, p.n, [p.hkv], [p.hd], precision=[dr.PRECISION_FP8])
    cache.store(0, dr.Pass(dev.ctx, range(p.n)), dev.put(p.k), dev.put(p.v))
    out = empty_rows(dev, p.q.size, bf16)
    dev.ctx.set_split(split)
    with wave_rows(dev, wave), rows_of(dev, bf16):
        try:
            cache.attention(0, [(put_rows(dev, p.q, bf16), out, dr.Pass(dev.ctx, p.pos))], p.h, sliding_window=window,
                            causal_prefix=prefix, scale=scale)
        finally:
            dev.ctx.set_split(0)
    got = dev.get(out.float()).reshape(p.q.shape)
    k, v = stored(p.k), stored(p.v)
    see = visible(p.n, p.pos, window, prefix)
    worst = 0.0
    for i in range(len(p.pos)):
        ki, vi = k[see[i]], v[see[i]]
        want, weighted = attend(p.q[i:i + 1], ki, vi, [0], scale)
        tol = bound(p.q[i:i + 1], ki, np.zeros_like(vi), weighted, want, scale, bf16) + weighted * p.n * 2.0 ** -24
        tol = tol + 2.0 ** -136 + (2.0 ** -134 if bf16 else 0.0) + (0.0 if more is None else more(i, see[i]))
        worst = max(worst, check(got[i:i + 1], want, tol, f"row {i}"))
    say(f"  {worst:.3f} of the bound")


# ---- rows of the smallest scale


@BF16
@SHAPES
@SMALL
def test_ordinary_values_after_the_smallest(dev, shape, size, bf16):
    """V rows of the smallest scale in the first tiles of every wave, ordinary ones
    after them: queries that see both, and some that see the small ones alone."""
    h, hkv, hd, wave = shape
    rng = np.random.default_rng(hd + wave)
    p = Problem(rng, h, hkv, hd, 600, [200, 210, 255, 300, 330, *range(580, 600)])
    p.v[:256] *= np.float32(size)
    assert (np.abs(p.v[:256]).max(-1) <= 1.75 * 2.0 ** -118).mean() > 0.9
    run(dev, p, wave, bf16)
    run(dev, p, wave, bf16, prefix=600)
    run(dev, p, wave, bf16, prefix=600, split=2)
    p.v = np.ascontiguousarray(p.v[::-1])
    run(dev, p, wave, bf16, prefix=600, split=3)


@BF16
@SHAPES
def test_keys_of_the_smallest_scale(dev, shape, bf16):
    """K rows of the smallest scale whose scores a large query makes ordinary, in
    tiles that they share with larger ones out of sight."""
    h, hkv, hd, wave = shape
    rng = np.random.default_rng(hd + wave + 1)
    p = Problem(rng, h, hkv, hd, 300, range(140, 200))
    p.q *= np.float32(2.0 ** 119)
    p.k *= np.float32(2.0 ** -120)
    assert np.abs(p.k).max() <= 1.75 * 2.0 ** -118
    run(dev, p, wave, bf16)
    p.k[:100] *= np.float32(2.0 ** 110)
    p.k[220:] *= np.float32(2.0 ** 110)
    run(dev, p, wave, bf16, window=20)
    run(dev, p, wave, bf16, window=20, split=2)


@BF16
@SHAPES
@pytest.mark.parametrize("size", [1e-34, 1e-35, 1.2e-36])
def test_small_outputs(dev, shape, size, bf16):
    """Nothing but V rows near the smallest numbers."""
    h, hkv, hd, wave = shape
    rng = np.random.default_rng(hd + wave + 2)
    p = Problem(rng, h, hkv, hd, 300, range(240, 300))
    p.v *= np.float32(size)
    run(dev, p, wave, bf16)
    run(dev, p, wave, bf16, window=100, split=3)


# ---- sizes that grow


@BF16
@SHAPES
def test_values_that_grow_in_steps(dev, shape, bf16):
    """V rows that grow 2^60 at a time, each step within what the accumulators
    stand: a query that sees the first of them alone keeps its bits beside one
    that sees them all."""
    h, hkv, hd, wave = shape
    rng = np.random.default_rng(hd + wave + 3)
    p = Problem(rng, h, hkv, hd, 1024, [10, 100, 255, 256, 500, 511, 700, 1023])
    p.v *= np.exp2(-100.0 + 60 * (np.arange(1024) // 256)).astype(np.float32)[:, None, None]
    run(dev, p, wave, bf16, prefix=1024)
    run(dev, p, wave, bf16, prefix=1024, split=1)


# ---- small queries


@BF16
@SHAPES
@pytest.mark.parametrize("e", [105, 113, 120])
def test_small_queries_of_large_keys(dev, shape, e, bf16):
    """Query rows around 2^-e, K rows around 2^e, and the other way round."""
    h, hkv, hd, wave = shape
    rng = np.random.default_rng(hd + wave + e)
    p = Problem(rng, h, hkv, hd, 200, range(150, 200))
    q, k = p.q, p.k
    p.q, p.k = q * np.float32(2.0 ** -e), k * np.float32(2.0 ** e)
    run(dev, p, wave, bf16)
    run(dev, p, wave, bf16, window=60, split=2)
    p.q, p.k = q * np.float32(2.0 ** e), k * np.float32(2.0 ** -e)
    run(dev, p, wave, bf16)


# ---- larger rows out of sight


@BF16
@SHAPES
def test_light_keys_beside_a_larger_row_out_of_sight(dev, shape, bf16):
    """One key takes almost all of a row's weight, the others, alike, about 2^-12
    of it; dims in which the heavy key's value is 0 are theirs alone.  In their
    tile lies a V row that no query sees, 2^12 times as large (bf16 rows 2^16).

    A weight times its scale, relative to the largest scale met, is rounded to
    f16 planes whose last bit is 2^-24: off by 2^-24 (two planes) or 2^-25, in
    units in which the row's largest weight is 2^10 at least.  So a key adds at
    most 2^-34 (2^-35) of its value times the ratio of the scales, over the sum
    of weights relative to the largest."""
    h, hkv, hd, wave = shape
    rng = np.random.default_rng(hd + wave + 4)
    p = Problem(rng, h, hkv, hd, 32, range(12, 31))
    ratio = 16 if bf16 else 12
    p.v = rng.uniform(-1, 1, p.v.shape).astype(np.float32)
    p.v[..., hd // 2] = 1.75  # (every row's largest: one scale)
    p.v[0, :, :hd // 2] = 0
    p.v[31] *= np.float32(2.0 ** ratio)
    p.k[:] = 0
    p.k[:, :, 1] = 1
    p.k[0, :, 0] = 8  # (a code, so that its score is known)
    p.q[:] = 0
    p.q[..., 0] = rng.uniform(0.9, 1.1, p.q.shape[:2]) * 12 * math.log(2) * math.sqrt(hd) / 8

    def more(i, seen):
        v = np.repeat(np.abs(stored(p.v)[seen]).sum(0), h // hkv, axis=0)[None]
        return v * 2.0 ** (ratio - (35 if bf16 else 34))

    run(dev, p, wave, bf16, prefix=32, more=more)


# ---- a scale that is no number


@BF16
@SHAPES
def test_nan_scale(dev, shape, bf16):
    """Scores that are NaN: every row is, as on the other layers."""
    h, hkv, hd, wave = shape
    rng = np.random.default_rng(hd + wave + 5)
    p = Problem(rng, h, hkv, hd, 70, range(40, 70))
    run(dev, p, wave, bf16, scale=math.nan)
    run(dev, p, wave, bf16, window=20, split=2, scale=math.nan)
