"""DR_PRECISION_FP8 cache layers: what a store leaves in them (every bit, through
the gather) against the format's definition in float64, at head dims that fill
no tile, runs and lists that start and end inside tiles, rows with zeros,
subnormals, NaN and infinities; the rows that a call does not name stay.
Needs an MI355X."""
from __future__ import annotations

import numpy as np
import pytest

import dr_attn as dr
from fp8_reference import stored

from test_gpu_parity import dev, say, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def layer(dev, n, hkv, hd, **kw):
    return dr.StepCache(dev.ctx, n, [hkv], [hd], precision=[dr.PRECISION_FP8], **kw)


def gather(dev, cache, p, n, hkv, hd, batch=0):
    k, v = dev.empty(n * hkv * hd), dev.empty(n * hkv * hd)
    cache.gather_pass(0, p, k, v, batch=batch)
    return dev.get(k).reshape(n, hkv, hd), dev.get(v).reshape(n, hkv, hd)


def rows(rng, n, hkv, hd):
    """Rows of many sizes, values of many sizes in them."""
    x = rng.standard_normal((n, hkv, hd)) * np.exp2(rng.integers(-9, 9, (n, hkv, hd)) * rng.random((n, hkv, 1)))
    return (x * np.exp2(rng.integers(-30, 30, (n, hkv, 1)))).astype(np.float32)


POSITIONS = {
    "one": lambda n: [n - 1],
    "first": lambda n: [0],
    "all": lambda n: range(n),
    "run": lambda n: range(n // 3, n - n // 5),
    "scattered": lambda n: sorted({0, 1, n - 1, *range(2, n, 3), *range(n // 2, n // 2 + 9)}),
    "even": lambda n: range(0, n, 2),
}


@pytest.mark.parametrize("hd", [1, 2, 20, 63, 64, 80, 128, 130, 200, 256, 300, 512])
@pytest.mark.parametrize("where", list(POSITIONS))
def test_store_and_gather(dev, hd, where):
    n, hkv = 101, 3
    rng = np.random.default_rng(hd * 7 + len(where))
    cache = layer(dev, n, hkv, hd)
    whole = dr.Pass(dev.ctx, range(n))
    K, V = rows(rng, n, hkv, hd), rows(rng, n, hkv, hd)
    cache.store(0, whole, dev.put(K), dev.put(V))
    pos = [p for p in POSITIONS[where](n)]
    k, v = rows(rng, len(pos), hkv, hd), rows(rng, len(pos), hkv, hd)
    cache.store(0, dr.Pass(dev.ctx, pos), dev.put(k), dev.put(v))
    K[pos], V[pos] = k, v
    for got, x in zip(gather(dev, cache, whole, n, hkv, hd), (K, V)):
        assert np.array_equal(got, stored(x).astype(np.float32))
    # the pass's own rows, and the host list in another order and twice
    for got, x in zip(gather(dev, cache, dr.Pass(dev.ctx, pos), len(pos), hkv, hd), (k, v)):
        assert np.array_equal(got, stored(x).astype(np.float32))
    order = rng.integers(0, n, 37)
    gk, gv = dev.empty(37 * hkv * hd), dev.empty(37 * hkv * hd)
    cache.gather(0, order, gk, gv)
    for got, x in ((gk, K), (gv, V)):
        assert np.array_equal(dev.get(got).reshape(37, hkv, hd), stored(x[order]).astype(np.float32))


def test_every_rounding(dev):
    """Every e4m3 code, the values half way between neighbours and one f32 step
    to either side of them, in rows whose largest value fixes the scale."""
    codes = np.array([(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1] + [m / 512 for m in range(8)])
    codes = np.unique(codes)
    mid = ((codes[1:] + codes[:-1]) / 2).astype(np.float32)
    x = np.concatenate([codes.astype(np.float32), mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(999))])
    x = x[x <= 448]
    x = np.concatenate([x, -x, np.zeros(-len(x) * 2 % 63, np.float32)]).reshape(-1, 63)
    for e, top in ((0, 448.0), (-100, 257.0), (90, 256.0)):
        r = np.concatenate([np.minimum(np.abs(x), top) * np.sign(x), np.full((len(x), 1), top, np.float32)], 1)
        r = np.ldexp(r.astype(np.float32), e).astype(np.float32).reshape(len(x), 1, 64)
        cache = layer(dev, len(r), 1, 64)
        p = dr.Pass(dev.ctx, range(len(r)))
        cache.store(0, p, dev.put(r), dev.put(-r))
        gk, gv = gather(dev, cache, p, len(r), 1, 64)
        assert np.array_equal(gk, stored(r).astype(np.float32)) and np.array_equal(gv, stored(-r).astype(np.float32))


def test_scale_borders(dev):
    """A row's largest value just at, below and above the borders of its scale,
    the largest f32, subnormals and zeros."""
    tops = []
    for e in (-149, -140, -127, -126, -120, -118, -117, 0, 100, 127):
        for m in (1.0, 1.5, 1.75, np.nextafter(np.float32(1.75), np.float32(2)), 1.9375, np.float32(2) - np.float32(2 ** -23)):
            t = np.float32(np.ldexp(np.float64(m), e))
            if np.isfinite(t):
                tops.append(t)
    tops = np.array(tops + [0.0], np.float32)
    for hd in (64, 128, 512):
        r = (np.linspace(-1, 1, hd)[None] * tops[:, None].astype(np.float64)).astype(np.float32)
        r[:, 3] = tops
        r = r.reshape(-1, 1, hd)
        cache = layer(dev, len(r), 1, hd)
        p = dr.Pass(dev.ctx, range(len(r)))
        cache.store(0, p, dev.put(r), dev.put(-r))
        gk, gv = gather(dev, cache, p, len(r), 1, hd)
        assert np.array_equal(gk, stored(r).astype(np.float32)) and np.array_equal(gv, stored(-r).astype(np.float32))


@pytest.mark.parametrize("hd", [64, 100, 512])
def test_nan_rows(dev, hd):
    """A NaN or an infinity makes its own row NaN and no other; storing the
    position again clears it."""
    rng = np.random.default_rng(hd)
    n, hkv = 70, 2
    k, v = rows(rng, n, hkv, hd), rows(rng, n, hkv, hd)
    k[3, 0, 5], k[40, 1, 0], k[69, 1, hd - 1] = np.nan, np.inf, -np.inf
    v[0, 0, 0], v[33, 1, 7], v[34, 0, hd - 1] = -np.inf, np.nan, np.inf
    cache = layer(dev, n, hkv, hd)
    p = dr.Pass(dev.ctx, range(n))
    cache.store(0, p, dev.put(k), dev.put(v))
    for got, x in zip(gather(dev, cache, p, n, hkv, hd), (k, v)):
        assert np.array_equal(got, stored(x).astype(np.float32), equal_nan=True)
        assert np.isnan(got).sum() == 3 * hd
    k, v = rows(rng, n, hkv, hd), rows(rng, n, hkv, hd)
    cache.store(0, p, dev.put(k), dev.put(v))
    for got, x in zip(gather(dev, cache, p, n, hkv, hd), (k, v)):
        assert np.array_equal(got, stored(x).astype(np.float32))


def test_never_stored_positions_are_zero(dev):
    cache = layer(dev, 50, 2, 128)
    p = dr.Pass(dev.ctx, range(50))
    for got in gather(dev, cache, p, 50, 2, 128):
        assert not got.any()


@pytest.mark.parametrize("precision", [dr.PRECISION_BF16, dr.PRECISION_HILO, dr.PRECISION_FP8])
@pytest.mark.parametrize("pos", [range(7, 61), [0, 3, 31, 32, 64]])
def test_gather_pass_is_gather(dev, precision, pos):
    """dr_cache_gather_pass gives what dr_cache_gather gives, at every precision."""
    n, hkv, hd = 65, 2, 100
    rng = np.random.default_rng(1)
    cache = dr.StepCache(dev.ctx, n, [hkv], [hd], n_batch=2, precision=[precision])
    for b in range(2):
        cache.store(0, dr.Pass(dev.ctx, range(n)), dev.put(rows(rng, n, hkv, hd)), dev.put(rows(rng, n, hkv, hd)), batch=b)
    size = len(pos) * hkv * hd
    for b in range(2):
        k, v = dev.empty(size), dev.empty(size)
        cache.gather(0, pos, k, v, batch=b)
        gk, gv = gather(dev, cache, dr.Pass(dev.ctx, pos), len(pos), hkv, hd, batch=b)
        assert np.array_equal(dev.get(k), gk.reshape(-1)) and np.array_equal(dev.get(v), gv.reshape(-1))


def test_layers_of_every_precision(dev):
    """A cache with a layer of each kind, and a layer that changes its kind: its
    rows are dropped to and from 8 bits, and what other layers hold stays."""
    n, hkv, hd = 40, 2, 64
    rng = np.random.default_rng(2)
    cache = dr.StepCache(dev.ctx, n, [hkv] * 3, [hd] * 3,
                         precision=[dr.PRECISION_BF16, dr.PRECISION_FP8, dr.PRECISION_HILO])
    p = dr.Pass(dev.ctx, range(n))
    x = rng.standard_normal((n, hkv, hd)).astype(np.float32)

    def get(l):
        k, v = dev.empty(x.size), dev.empty(x.size)
        cache.gather_pass(l, p, k, v)
        k, v = dev.get(k), dev.get(v)
        assert np.array_equal(k, v)
        return k.reshape(x.shape)

    for l in range(3):
        cache.store(l, p, dev.put(x), dev.put(x))
    bf, f8, hi = (get(l) for l in range(3))
    assert np.abs(bf - x).max() <= 2.0 ** -8 * np.abs(x).max() and np.abs(hi - x).max() <= 2.0 ** -16 * np.abs(x).max()
    assert np.array_equal(f8, stored(x).astype(np.float32))
    cache.set_precision(1, dr.PRECISION_FP8)  # nothing changes
    assert np.array_equal(get(1), f8)
    cache.set_precision(1, dr.PRECISION_HILO)
    assert not get(1).any()
    cache.store(1, p, dev.put(x), dev.put(x))
    assert np.array_equal(get(1), hi)
    cache.set_precision(1, dr.PRECISION_FP8)
    assert not get(1).any()
    cache.store(1, p, dev.put(x), dev.put(x))
    assert np.array_equal(get(1), f8) and np.array_equal(get(0), bf) and np.array_equal(get(2), hi)


def test_refusals(dev):
    cache = layer(dev, 40, 2, 64)
    p = dr.Pass(dev.ctx, range(40))
    x = dev.empty(40 * 2 * 64)

    def refused(status, call, *args):
        with pytest.raises(dr.DrError) as e:
            call(*args)
        assert e.value.status == status, e.value

    bad = dr.DR_ERR_INVALID
    refused(bad, cache.gather_pass, 1, p, x, x)  # no layer 1
    refused(bad, cache.gather_pass, 0, p, None, x)
    refused(bad, cache.gather_pass, 0, p, x, None)
    refused(bad, cache.gather_pass, 0, dr.Pass(dev.ctx, [40]), x, x)  # position 40 of 40
    refused(bad, cache.gather_pass, 0, dr.Pass(dr.Context(0), [0]), x, x)
    refused(bad, cache.set_precision, 0, 3)
    with pytest.raises(dr.DrError):
        dr.StepCache(dev.ctx, 40, [2], [64], precision=[3])
    cache.gather_pass(0, dr.Pass(dev.ctx, []), None, None)  # no rows: nothing to do


def test_planes_past_32_bit_offsets(dev):
    """A plane of 4.4 GB: its last head's and first head's rows, at both ends."""
    n, hkv, hd = 1 << 20, 33, 128
    cache = layer(dev, n, hkv, hd)
    rng = np.random.default_rng(3)
    for pos in ([0, 1, n - 2, n - 1], range(n - 40, n), range(31, 65)):
        p = dr.Pass(dev.ctx, pos)
        k, v = rows(rng, len(pos), hkv, hd), rows(rng, len(pos), hkv, hd)
        cache.store(0, p, dev.put(k), dev.put(v))
        for got, x in zip(gather(dev, cache, p, len(pos), hkv, hd), (k, v)):
            assert np.array_equal(got, stored(x).astype(np.float32))
