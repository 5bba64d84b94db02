"""The launch shapes of attention over DR_PRECISION_FP8 layers: 16 and 32 rows a
wave (at head dims 257-512 the 64-row kernel whose waves split the head dim),
forced and as the planner picks them, joins of few and many key splits, and
stores that go tile by tile.  The same bounds as the 8 bit attention's other
tests.  Needs an MI355X."""
from __future__ import annotations

import math

import numpy as np
import pytest

import dr_attn as dr
from fp8_reference import attend, bound, check, stored

from test_gpu_fp8_attention import Problem, empty_rows, put_rows, rows_of, run
from test_gpu_parity import dev, say, torch  # noqa: F401

pytestmark = pytest.mark.gpu

ROWS = pytest.mark.parametrize("rows", [16, 32])
BF16 = pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])


class wave_rows:
    """16 or 32 query rows a wave within a block."""

    def __init__(self, dev, rows):
        self.ctx, self.rows = dev.ctx, rows

    def __enter__(self):
        self.ctx.set_wave_rows(self.rows)

    def __exit__(self, *a):
        self.ctx.set_wave_rows(0)


# (query heads, KV heads, head dim, keys, active positions, window, prefix, key splits)
CASES = {
    "one_key": (1, 1, 512, 1, [0], None, None, 0),
    "one_row": (2, 1, 512, 33, [32], None, None, 0),
    "two_tiles": (2, 2, 512, 64, range(64), None, None, 1),
    "64_rows": (4, 2, 512, 161, range(100, 132), None, None, 1),
    "65_rows": (1, 1, 512, 161, range(96, 161), None, None, 1),
    "split_2": (3, 1, 512, 161, range(100, 161), None, None, 2),
    "split_3": (4, 2, 512, 300, range(0, 300, 7), None, None, 3),
    "split_6": (4, 2, 512, 300, range(230, 300), None, None, 6),
    "more_splits_than_tiles": (4, 1, 512, 70, range(30, 70), None, None, 9),
    "causal": (2, 1, 512, 150, range(150), None, 150, 1),
    "causal_split": (2, 1, 512, 150, range(150), None, 121, 2),
    "window": (2, 1, 512, 200, range(40, 150), 33, None, 1),
    "window_1": (1, 1, 512, 70, range(70), 1, None, 0),
    "window_causal_scattered": (6, 2, 512, 300, [0, 1, 31, 32, 63, 64, 65, 100, 220, 221, 222, 255, 298, 299], 120, 200, 0),
    "hd_257": (2, 2, 257, 97, range(30, 97), None, None, 0),
    "hd_300": (3, 1, 300, 130, range(60, 130), None, 100, 2),
    "hd_500": (8, 2, 500, 130, range(100, 130), 50, None, 1),
    "hd_128": (4, 2, 128, 300, range(250, 300), None, 290, 1),
    "hd_128_split_5": (4, 2, 128, 400, range(380, 400), None, None, 5),
    "hd_64_split_20": (4, 1, 64, 700, range(680, 700), None, None, 20),
    "hd_80": (6, 3, 80, 321, range(0, 321, 5), 64, None, 3),
}


@BF16
@ROWS
@pytest.mark.parametrize("name", list(CASES))
def test_rows_of_a_wave(dev, name, rows, bf16):
    h, hkv, hd, n, pos, window, prefix, split = CASES[name]
    rng = np.random.default_rng(sum(map(ord, name)))
    with wave_rows(dev, rows):
        info = run(dev, [Problem(rng, h, hkv, hd, n, pos)], window, prefix, bf16, split)
    assert info["rows_per_wave"] == rows and info["row_blocks"] == (2 if hd > 256 and rows == 32 else 1)


@BF16
@pytest.mark.parametrize("rows", [1, 40])
def test_scales_far_apart(dev, rows, bf16):
    """The largest V scale rises late in the walk, K's scales lie up to 2^12 apart."""
    rng = np.random.default_rng(rows)
    p = Problem(rng, 4, 2, 512, 450, range(450 - rows, 450), spread=4.0)
    p.v = p.v[np.argsort(np.abs(p.v).max((1, 2)))]
    with wave_rows(dev, 32):
        run(dev, [p], bf16=bf16, split=1)
        run(dev, [p], bf16=bf16, split=3)


@BF16
def test_growing_scores(dev, bf16):
    """Scores that keep rising along the keys move the running maximum again and
    again, in one row block more than in the other; in the other slot they fall."""
    rng = np.random.default_rng(1)
    up, down = (Problem(rng, 4, 2, 512, 700, range(660, 700)) for _ in range(2))
    ramp = np.linspace(0.0, 1.0, 700, dtype=np.float32)[:, None, None]
    up.k = np.abs(up.k) * ramp
    down.k = np.abs(down.k) * ramp[::-1]
    up.q, down.q = np.abs(up.q) * 3, np.abs(down.q) * 3
    up.q[:8] *= 0.05
    down.q[8:] *= 0.05
    with wave_rows(dev, 32):
        run(dev, [up, down], bf16=bf16, split=1)
        run(dev, [up, down], bf16=bf16, split=2)


def test_slots_of_different_lengths(dev):
    rng = np.random.default_rng(2)
    probs = [Problem(rng, 4, 2, 512, 200, pos) for pos in ([], range(60, 200), [3], range(0, 200, 7))]
    with wave_rows(dev, 32):
        for bf16 in (False, True):
            run(dev, probs, window=90, bf16=bf16)
            run(dev, probs, prefix=120, bf16=bf16, split=3)


def test_empty_window_is_nan(dev):
    rng = np.random.default_rng(3)
    with wave_rows(dev, 32):
        run(dev, [Problem(rng, 4, 2, 512, 70, range(30, 70))], window=0)
        run(dev, [Problem(rng, 4, 2, 512, 70, range(30, 70))], window=0, split=2)


@BF16
def test_nan_and_infinities_in_and_out_of_sight(dev, bf16):
    """Cache rows with a NaN or an infinity reach the queries that see them and no
    others, though they share tiles; a query row's NaN stays its own."""
    rng = np.random.default_rng(4)
    n, hd, pos = 160, 512, list(range(10, 74))
    p = Problem(rng, 4, 2, hd, n, pos)
    p.k[60, 0, 1], p.k[62, 1, 0] = np.nan, np.inf
    p.v[100, 0, hd - 1], p.v[41, 1, 3], p.v[0, 0, 0] = -np.inf, np.nan, np.nan
    with wave_rows(dev, 32):
        run(dev, [p], prefix=n, bf16=bf16)
        run(dev, [p], window=12, bf16=bf16)
        run(dev, [p], window=30, prefix=50, bf16=bf16, split=2)
        p.q[5, 1, 2], p.q[9, 3, 0] = np.nan, np.inf
        got = np.isnan(attend(np.where(np.isfinite(p.q), p.q, 0), stored(p.k), stored(p.v), pos, 0.04, 12)[0])
        cache = dr.StepCache(dev.ctx, n, [2], [hd], precision=[dr.PRECISION_FP8])
        cache.store(0, dr.Pass(dev.ctx, range(n)), dev.put(p.k), dev.put(p.v))
        out = empty_rows(dev, p.q.size, bf16)
        with rows_of(dev, bf16):
            cache.attention(0, [(put_rows(dev, p.q, bf16), out, dr.Pass(dev.ctx, pos))], 4, sliding_window=12, scale=0.04)
    got[5, 1], got[9, 3] = True, True
    assert np.array_equal(np.isnan(dev.get(out.float())).reshape(got.shape), got)


def test_the_planner_takes_the_wide_kernel(dev):
    """More 16-row blocks than CUs: without any forced shape, rows that fill no
    block, and the same bits from a repeated call."""
    rng = np.random.default_rng(5)
    p = Problem(rng, 32, 16, 512, 150, range(7, 150))
    for bf16 in (False, True):
        assert run(dev, [p], prefix=130, bf16=bf16)["row_blocks"] == 2
    cache = dr.StepCache(dev.ctx, p.n, [p.hkv], [p.hd], precision=[dr.PRECISION_FP8])
    cache.store(0, dr.Pass(dev.ctx, range(p.n)), dev.put(p.k), dev.put(p.v))
    outs = [dev.empty(p.q.size) for _ in range(2)]
    for split in (0, 3):
        dev.ctx.set_split(split)
        try:
            for o in outs:
                cache.attention(0, [(dev.put(p.q), o, dr.Pass(dev.ctx, p.pos))], p.h, scale=0.04, noalloc=o is outs[1])
        finally:
            dev.ctx.set_split(0)
        assert dev.ctx.last_launch()["row_blocks"] == 2
        assert np.array_equal(dev.get(outs[0]), dev.get(outs[1]))


@pytest.mark.parametrize("h,hkv,hd,n,rows", [(8, 1, 512, 1500, 6), (16, 2, 256, 3000, 8), (28, 4, 128, 3000, 5),
                                             (8, 2, 64, 3000, 20), (4, 4, 128, 3000, 1)])
def test_the_planner_splits_long_keys(dev, h, hkv, hd, n, rows):
    """Few rows over many keys: the planner's own splits."""
    rng = np.random.default_rng(n + hd)
    assert run(dev, [Problem(rng, h, hkv, hd, n, range(n - rows, n))])["n_split"] > 1


def test_captured_wide_call_replays(dev):
    """A split call of the 64-row kernel in a hipGraph: its tickets are ready again
    for every replay and for the eager calls between them."""
    t = dev.t
    rng = np.random.default_rng(6)
    n, h, hkv, hd, m = 200, 4, 2, 512, 60
    cache = dr.StepCache(dev.ctx, n, [hkv], [hd], precision=[dr.PRECISION_FP8])
    K = rng.standard_normal((n, hkv, hd)).astype(np.float32)
    cache.store(0, dr.Pass(dev.ctx, range(n)), dev.put(K), dev.put(K))
    p, q = dr.Pass(dev.ctx, range(n - m, n)), dev.put(rng.standard_normal(m * h * hd).astype(np.float32))
    out, eager = dev.empty(m * h * hd), dev.empty(m * h * hd)
    dev.ctx.set_split(3)
    with wave_rows(dev, 32):
        try:
            cache.attention(0, [(q, out, p)], h, scale=0.04)
            dev.stream.synchronize()
            graph = t.cuda.CUDAGraph()
            with t.cuda.graph(graph, stream=dev.stream):
                cache.attention(0, [(q, out, p)], h, scale=0.04)
            for i in range(4):
                with t.cuda.stream(dev.stream):
                    q.mul_(0.9)
                    out.zero_()
                    graph.replay()
                cache.attention(0, [(q, eager, p)], h, scale=0.04)
                assert np.array_equal(dev.get(out), dev.get(eager))
        finally:
            dev.ctx.set_split(0)


@pytest.mark.parametrize("precision", [dr.PRECISION_HILO, dr.PRECISION_BF16])
def test_forced_fp8_means_auto_on_other_layers(dev, precision):
    """The 8 bit family forced leaves a hi/lo layer its f32-accurate kernel."""
    rng = np.random.default_rng(7)
    n, h, hkv, hd = 90, 4, 2, 128
    cache = dr.StepCache(dev.ctx, n, [hkv], [hd], precision=[precision])
    p = dr.Pass(dev.ctx, range(n))
    k, v, q = (dev.put(rng.standard_normal(n * c * hd).astype(np.float32)) for c in (hkv, hkv, h))
    cache.store(0, p, k, v)
    outs = [dev.empty(n * h * hd) for _ in range(2)]
    kinds = []
    for kernel, o in zip((dr.KERNEL_AUTO, dr.KERNEL_FP8), outs):
        dev.ctx.set_kernel(kernel)
        try:
            cache.attention(0, [(q, o, p)], h, scale=0.09)
        finally:
            dev.ctx.set_kernel(dr.KERNEL_AUTO)
        kinds.append(dev.ctx.last_launch()["kernel"])
    assert kinds[0] == kinds[1] and (kinds[0] == dr.KERNEL_HILO) == (precision == dr.PRECISION_HILO)
    assert np.array_equal(dev.get(outs[0]), dev.get(outs[1]))


# ---- stores: long runs go tile by tile, very long ones past the caches


def gather(dev, cache, p, n, hkv, hd):
    k, v = dev.empty(n * hkv * hd), dev.empty(n * hkv * hd)
    cache.gather_pass(0, p, k, v)
    return k, v


@pytest.mark.parametrize("hkv,hd", [(1, 20), (2, 64), (1, 128), (2, 130)])
@pytest.mark.parametrize("first,last", [(0, 4200), (1, 4199), (31, 4129), (32, 4160)])
def test_store_tile_by_tile(dev, hkv, hd, first, last):
    """Runs of more than a hundred tiles that start and end inside tiles."""
    n = 4200
    rng = np.random.default_rng(hd + first)
    K, V = (rng.standard_normal((n, hkv, hd)).astype(np.float32) * np.float32(2.0) ** rng.integers(-9, 9, (n, 1, 1))
            for _ in range(2))
    K, V = K.astype(np.float32), V.astype(np.float32)
    cache = dr.StepCache(dev.ctx, n, [hkv], [hd], precision=[dr.PRECISION_FP8])
    whole = dr.Pass(dev.ctx, range(n))
    cache.store(0, whole, dev.put(K), dev.put(V))
    k, v = (rng.standard_normal((last - first, hkv, hd)).astype(np.float32) for _ in range(2))
    cache.store(0, dr.Pass(dev.ctx, range(first, last)), dev.put(k), dev.put(v))
    K[first:last], V[first:last] = k, v
    for got, x in zip(gather(dev, cache, whole, n, hkv, hd), (K, V)):
        assert np.array_equal(dev.get(got).reshape(x.shape), stored(x).astype(np.float32))


def test_store_past_the_caches(dev):
    """A store of more than 2^24 values in one call, against the same rows in
    scattered lists, bit for bit; a sample of them against the format."""
    t = dev.t
    n, hkv, hd = 4111, 8, 512
    assert n * hkv * hd > 1 << 24
    rng = np.random.default_rng(8)
    with t.cuda.stream(dev.stream):
        gen = t.Generator(device="cuda").manual_seed(8)
        K, V = (t.randn(n, hkv, hd, device="cuda", generator=gen) for _ in range(2))
    one, lists = (dr.StepCache(dev.ctx, n, [hkv], [hd], precision=[dr.PRECISION_FP8]) for _ in range(2))
    whole = dr.Pass(dev.ctx, range(n))
    one.store(0, whole, K, V)
    for part in np.array_split(rng.permutation(n), 3):
        part = np.sort(part)
        with t.cuda.stream(dev.stream):
            rows = t.from_numpy(part).cuda()
            k, v = K[rows].contiguous(), V[rows].contiguous()
        lists.store(0, dr.Pass(dev.ctx, part.tolist()), k, v)
        dev.stream.synchronize()
    a, b = gather(dev, one, whole, n, hkv, hd), gather(dev, lists, whole, n, hkv, hd)
    dev.stream.synchronize()
    for x, y, z in zip(a, b, (K, V)):
        assert bool((x == y).all())
        some = rng.integers(0, n, 40)
        assert np.array_equal(dev.get(x).reshape(n, hkv, hd)[some], stored(dev.get(z)[some]).astype(np.float32))
