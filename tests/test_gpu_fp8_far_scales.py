"""Attention over DR_PRECISION_FP8 layers whose rows' scales lie far apart: huge
rows that a query does not see must not cost it bits, whatever tile they share,
and of those that it sees a row's largest product is the measure of its error.
Positions that were never stored read as zeros.  Needs an MI355X."""
from __future__ import annotations

import math

import numpy as np
import pytest

import dr_attn as dr
from fp8_reference import attend, bound, check, stored
from helpers import bf16_round

from test_gpu_fp8_attention import Problem, empty_rows, put_rows, rows_of
from test_gpu_fp8_wide import wave_rows
from test_gpu_parity import dev, say, torch  # noqa: F401

pytestmark = pytest.mark.gpu

BF16 = pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
# (query heads, KV heads, head dim, rows a wave)
SHAPES = pytest.mark.parametrize("shape", [(4, 2, 64, 32), (4, 2, 64, 16), (4, 2, 128, 32), (4, 2, 128, 16), (4, 2, 256, 16),
                                           (4, 2, 512, 16), (4, 2, 512, 32), (6, 3, 80, 32)], ids=str)


def visible(n, pos, window, prefix):
    p, j = np.asarray(pos)[:, None], np.arange(n)[None, :]
    see = np.ones((len(pos), n), bool)
    if window is not None:
        see &= np.abs(p - j) < window
    if prefix is not None:
        see &= ~((p < prefix) & (j > p))
    return see


def run(dev, p, wave, bf16, window=None, prefix=None, split=0, store=None):
    """A call checked row by row, each against the bound of the keys that it sees.
    Its last term, an absolute step, is taken of the row's own largest product:
    2^-25 in units where that row's largest weight is at least 1/2."""
    scale = 1 / math.sqrt(p.hd)
    if bf16:
        p.q = bf16_round(p.q)
    cache = dr.StepCache(dev.ctx, p.n, [p.hkv], [p.hd], precision=[dr.PRECISION_FP8])
    store = list(range(p.n)) if store is None else store
    cache.store(0, dr.Pass(dev.ctx, store), dev.put(p.k[store]), dev.put(p.v[store]))
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
    gone = np.setdiff1d(np.arange(p.n), store)
    k[gone], v[gone] = 0, 0
    see = visible(p.n, p.pos, window, prefix)
    worst = 0.0
    for i in range(len(p.pos)):
        ki, vi = k[see[i]], v[see[i]]
        want, weighted = attend(p.q[i:i + 1], ki, vi, [0], scale)
        tol = bound(p.q[i:i + 1], ki, np.zeros_like(vi), weighted, want, scale, bf16) + weighted * p.n * 2.0 ** -24
        worst = max(worst, check(got[i:i + 1], want, tol, f"row {i}"))
    say(f"  {worst:.3f} of the bound")


@BF16
@SHAPES
@pytest.mark.parametrize("size", [1e30, 1e6, 1e-30])
def test_rows_out_of_sight(dev, shape, size, bf16):
    """Rows of another size where no query, or only some, can see them: in front,
    behind, and within tiles that they share."""
    h, hkv, hd, wave = shape
    rng = np.random.default_rng(hd + wave)
    n, pos = 300, list(range(150, 190))
    p = Problem(rng, h, hkv, hd, n, pos)
    for at in ([0, 5, 100, 120], [225, 230, 250, 299]):
        p.k[at] *= np.float32(size)
        p.v[at] *= np.float32(size)
    run(dev, p, wave, bf16, window=25)
    run(dev, p, wave, bf16, window=25, split=2)
    p = Problem(rng, h, hkv, hd, n, pos)
    p.v[165] *= np.float32(size)  # (seen by half of the rows, its weight an ordinary one)
    p.v[170, 0] *= np.float32(size)
    run(dev, p, wave, bf16, prefix=n)
    run(dev, p, wave, bf16, window=20, prefix=180, split=3)


@BF16
@SHAPES
def test_rows_far_apart_in_sight(dev, shape, bf16):
    """V rows 2^+-40 of each other, K rows down to 2^-50."""
    h, hkv, hd, wave = shape
    rng = np.random.default_rng(hd + wave + 1)
    p = Problem(rng, h, hkv, hd, 333, range(290, 333))
    p.v *= np.exp2(rng.integers(-40, 41, (333, hkv, 1))).astype(np.float32)
    p.k *= np.exp2(rng.integers(-50, 1, (333, hkv, 1))).astype(np.float32)
    run(dev, p, wave, bf16)
    run(dev, p, wave, bf16, window=40, split=2)
    p.v = np.sort(np.abs(p.v), axis=0)  # growing along the keys
    run(dev, p, wave, bf16)
    p.v = np.ascontiguousarray(p.v[::-1])
    run(dev, p, wave, bf16, prefix=320)


@BF16
@SHAPES
def test_scores_that_grow_past_huge_values(dev, shape, bf16):
    """Huge V rows early, whose weights a later key's score makes negligible."""
    h, hkv, hd, wave = shape
    rng = np.random.default_rng(hd + wave + 2)
    p = Problem(rng, h, hkv, hd, 200, range(180, 200))
    p.q = np.abs(p.q)
    p.k = np.abs(p.k) * np.linspace(-9, 9, 200, dtype=np.float32)[:, None, None]
    p.v[:20] *= np.float32(2.0 ** 90)
    run(dev, p, wave, bf16)


@BF16
@SHAPES
def test_positions_never_stored(dev, shape, bf16):
    """They read as zeros: a first tile without a row, holes, rows that see nothing
    else, zeros that were stored."""
    h, hkv, hd, wave = shape
    rng = np.random.default_rng(hd + wave + 3)
    n = 170
    p = Problem(rng, h, hkv, hd, n, range(3, 120, 3))
    p.k[130:140], p.v[130:140] = 0, 0
    store = [i for i in range(40, n) if i % 7]
    run(dev, p, wave, bf16, store=store)
    run(dev, p, wave, bf16, prefix=n, store=store)
    run(dev, p, wave, bf16, window=12, store=store)
    run(dev, p, wave, bf16, window=12, prefix=60, store=store, split=2)


@BF16
@SHAPES
@pytest.mark.parametrize("size", [1e35, 1e-33])
def test_the_ends_of_the_range(dev, shape, size, bf16):
    """Outputs near the largest and the smallest numbers: rows of that size, sums
    of a few hundred weights over them."""
    h, hkv, hd, wave = shape
    rng = np.random.default_rng(hd + wave + 4)
    p = Problem(rng, h, hkv, hd, 260, range(200, 240))
    p.v *= np.float32(size)
    run(dev, p, wave, bf16)
    run(dev, p, wave, bf16, prefix=230, split=3)
    run(dev, p, wave, bf16, window=1)
