"""Attention over DR_PRECISION_FP8 cache layers against its definition in float64
on the values that the layer holds: head dims that fill no tile, grouped heads,
one key and one query up to several row blocks and key splits, scattered rows,
masks that end inside tiles or leave a row empty, NaN rows in and out of sight,
scales far apart, f32 and bf16 rows.  Bounds: fp8_reference.bound (rounding
steps of what the kernel holds in fewer bits).  Needs an MI355X."""
from __future__ import annotations

import math

import numpy as np
import pytest

import dr_attn as dr
import oracle as orc
from fp8_reference import attend, bound, check, stored
from helpers import bf16_round

from test_gpu_parity import dev, say, torch  # noqa: F401

pytestmark = pytest.mark.gpu


class Problem:
    """One slot's rows and an 8 bit layer that holds them."""

    def __init__(self, rng, h, hkv, hd, n, pos, spread=0.0):
        self.h, self.hkv, self.hd, self.n, self.pos = h, hkv, hd, n, list(pos)
        self.k, self.v = (rng.standard_normal((n, hkv, hd)).astype(np.float32) for _ in range(2))
        if spread:
            self.k *= np.exp2(-np.abs(rng.standard_normal((n, hkv, 1)) * spread)).astype(np.float32)
            self.v *= np.exp2(rng.standard_normal((n, hkv, 1)) * spread).astype(np.float32)
        self.q = rng.standard_normal((len(self.pos), h, hd)).astype(np.float32)


def put_rows(dev, x, bf16):
    return dev.put(x).to(dev.t.bfloat16) if bf16 else dev.put(x)


class rows_of:
    """The context's row type within a block."""

    def __init__(self, dev, bf16):
        self.ctx, self.t = dev.ctx, dr.DTYPE_BF16 if bf16 else dr.DTYPE_F32

    def __enter__(self):
        self.ctx.set_q_dtype(self.t)
        self.ctx.set_o_dtype(self.t)

    def __exit__(self, *a):
        self.ctx.set_q_dtype(dr.DTYPE_F32)
        self.ctx.set_o_dtype(dr.DTYPE_F32)


def empty_rows(dev, n, bf16):
    with dev.t.cuda.stream(dev.stream):
        return dev.t.full((n,), float("nan"), dtype=dev.t.bfloat16 if bf16 else dev.t.float32, device="cuda")


def run(dev, probs, window=None, prefix=None, bf16=False, split=0, scale=None, noalloc=False, kernel=0):
    """Attention of a batch of problems, checked slot by slot; the launch."""
    p0 = probs[0]
    scale = 1.0 / math.sqrt(p0.hd) if scale is None else scale
    cache = dr.StepCache(dev.ctx, p0.n, [p0.hkv], [p0.hd], n_batch=len(probs), precision=[dr.PRECISION_FP8])
    items = []
    for b, p in enumerate(probs):
        if bf16:
            p.q = bf16_round(p.q)
        cache.store(0, dr.Pass(dev.ctx, range(p.n)), dev.put(p.k), dev.put(p.v), batch=b)
        items.append((put_rows(dev, p.q, bf16), empty_rows(dev, p.q.size, bf16), dr.Pass(dev.ctx, p.pos)))
    dev.ctx.set_split(split)
    dev.ctx.set_kernel(kernel)
    try:
        with rows_of(dev, bf16):
            cache.attention(0, items, p0.h, sliding_window=window, causal_prefix=prefix, scale=scale, noalloc=noalloc)
        info = dev.ctx.last_launch()
    finally:
        dev.ctx.set_split(0)
        dev.ctx.set_kernel(dr.KERNEL_AUTO)
    assert info["kernel"] == dr.KERNEL_FP8
    if split:
        assert info["n_split"] == split
    for b, p in enumerate(probs):
        k, v = stored(p.k), stored(p.v)
        want, weighted = attend(p.q, k, v, p.pos, scale, window, prefix)
        worst = check(dev.get(items[b][1].float()), want, bound(p.q, k, v, weighted, want, scale, bf16), f"slot {b}")
        say(f"  slot {b}: {worst:.3f} of the bound, {info['n_split']} splits")
    return info


# (query heads, KV heads, head dim, keys, active positions, window, prefix, key splits)
CASES = {
    "one_key": (1, 1, 64, 1, [0], None, None, 0),
    "one_row_of_33": (4, 1, 128, 33, [32], None, None, 0),
    "one_row_of_1000": (8, 2, 128, 1000, [500], None, None, 0),
    "one_row_split": (8, 2, 128, 1000, [999], None, None, 7),
    "more_splits_than_tiles": (2, 2, 128, 70, [5, 60], None, None, 9),
    "group_of_16": (16, 1, 128, 77, [76], None, None, 0),
    "17_packed_rows": (17, 1, 128, 300, [4], None, None, 0),
    "hd_1": (2, 1, 1, 40, range(40), None, None, 0),
    "hd_20": (6, 2, 20, 65, range(40, 65), None, None, 0),
    "hd_64": (8, 2, 64, 517, range(400, 517), None, None, 0),
    "hd_80": (6, 3, 80, 321, range(0, 321, 2), None, None, 0),
    "hd_80_one": (6, 3, 80, 321, [7], None, None, 3),
    "hd_128_mha": (4, 4, 128, 768, range(512, 768), None, None, 0),
    "hd_128_gqa_7": (28, 4, 128, 203, range(150, 203), None, None, 0),
    "hd_200": (4, 2, 200, 130, range(90, 130), None, None, 0),
    "hd_256": (4, 2, 256, 333, range(300, 333), None, None, 0),
    "hd_256_one": (4, 2, 256, 700, [699], None, None, 0),
    "hd_300": (2, 1, 300, 97, range(60, 97), None, None, 2),
    "hd_512": (4, 2, 512, 161, range(100, 161), None, None, 0),
    "hd_512_one": (8, 1, 512, 600, [0], None, None, 0),
    "all_causal": (4, 2, 128, 300, range(300), None, 300, 0),
    "causal_64": (8, 2, 64, 200, range(200), None, 150, 0),
    "causal_256": (2, 1, 256, 150, range(150), None, 121, 0),
    "causal_512": (2, 2, 512, 100, range(100), None, 70, 2),
    "prefix_0": (2, 2, 128, 64, range(64), None, 0, 0),
    "window": (4, 2, 128, 500, range(200, 330), 48, None, 0),
    "window_1": (4, 2, 128, 100, range(100), 1, None, 0),
    "window_2_scattered": (4, 2, 64, 300, [0, 31, 32, 33, 64, 150, 299], 2, None, 0),
    "window_causal": (4, 2, 128, 333, range(333), 64, 301, 0),
    "window_split": (4, 2, 128, 600, range(300, 310), 130, None, 4),
    "window_256": (4, 2, 256, 400, range(350, 400), 100, None, 0),
    "window_wide": (2, 2, 128, 90, range(40, 90), 100000, None, 0),
    "scattered": (4, 4, 128, 400, [0, 1, 5, 31, 32, 100, 163, 255, 256, 398, 399], 120, 200, 0),
    "group_spans_blocks": (20, 2, 128, 130, range(100, 130), 40, 110, 0),
    "rows_one_past_a_block": (2, 2, 128, 400, range(303, 400), None, None, 0),
    "many_blocks_causal": (8, 8, 128, 1500, range(1500), None, 1400, 0),
    "many_blocks_64_window": (16, 8, 64, 900, range(0, 900, 2), 33, None, 0),
}


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("name", list(CASES))
def test_against_definition(dev, name, bf16):
    h, hkv, hd, n, pos, window, prefix, split = CASES[name]
    rng = np.random.default_rng(sum(map(ord, name)))
    run(dev, [Problem(rng, h, hkv, hd, n, pos)], window, prefix, bf16, split)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("rows", [1, 40])
def test_scales_far_apart(dev, hd, rows, bf16):
    """K rows down to 2^-12 of the largest, V rows 2^+-12: the largest scale rises
    late in the walk, and early tiles are far below it."""
    rng = np.random.default_rng(hd + rows)
    p = Problem(rng, 4, 2, hd, 450, range(450 - rows, 450), spread=4.0)
    order = np.argsort(np.abs(p.v).max((1, 2)))
    p.v = p.v[order]
    run(dev, [p], bf16=bf16)


@pytest.mark.parametrize("hd", [128, 256])
def test_growing_scores(dev, hd):
    """Scores that keep rising along the keys move the running maximum again and
    again; then a batch in which they fall."""
    rng = np.random.default_rng(hd)
    up, down = (Problem(rng, 4, 2, hd, 700, range(660, 700)) for _ in range(2))
    ramp = np.linspace(0.0, 1.0, 700, dtype=np.float32)[:, None, None]
    up.k = np.abs(up.k) * ramp
    down.k = np.abs(down.k) * ramp[::-1]
    up.q, down.q = np.abs(up.q) * 3, np.abs(down.q) * 3
    run(dev, [up, down])


def test_slots_of_different_lengths(dev):
    rng = np.random.default_rng(5)
    probs = [Problem(rng, 8, 2, 128, 260, pos) for pos in ([], range(100, 260), [3], range(0, 260, 7))]
    for bf16 in (False, True):
        run(dev, probs, window=90, bf16=bf16)
        run(dev, probs, prefix=120, bf16=bf16, split=3)


@pytest.mark.parametrize("hd", [64, 128, 512])
def test_empty_window_is_nan(dev, hd):
    """A window of 0 lets no row see anything: NaN, as the reference's 0 * (1/0)."""
    rng = np.random.default_rng(hd)
    run(dev, [Problem(rng, 4, 2, hd, 70, range(30, 70))], window=0)
    run(dev, [Problem(rng, 4, 2, hd, 70, range(30, 70))], window=0, split=2)


@pytest.mark.parametrize("bf16", [False, True], ids=["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("rows", [1, 64])
def test_nan_and_infinities_in_and_out_of_sight(dev, hd, rows, bf16):
    """Rows of the cache with a NaN or an infinity reach the queries that see
    them, and no others, though they share tiles."""
    rng = np.random.default_rng(hd * 3 + rows)
    n = 160
    pos = [20] if rows == 1 else list(range(10, 74))
    p = Problem(rng, 4, 2, hd, n, pos)
    p.k[60, 0, 1], p.k[62, 1, 0] = np.nan, np.inf
    p.v[100, 0, hd - 1], p.v[41, 1, 3], p.v[0, 0, 0] = -np.inf, np.nan, np.nan
    # (a causal prefix: position 20 sees 0..20; later rows see 41, 60 and 62)
    run(dev, [p], prefix=n, bf16=bf16)
    run(dev, [p], window=12, bf16=bf16)
    run(dev, [p], window=30, prefix=50, bf16=bf16, split=2)
    if rows > 1:
        q = p.q.copy()
        p.q[5, 1, 2], p.q[9, 3, 0] = np.nan, np.inf  # a query row of its own
        got = np.isnan(attend(np.where(np.isfinite(p.q), p.q, 0), stored(p.k), stored(p.v), pos, 0.08, 12)[0])
        cache = dr.StepCache(dev.ctx, n, [2], [hd], precision=[dr.PRECISION_FP8])
        cache.store(0, dr.Pass(dev.ctx, range(n)), dev.put(p.k), dev.put(p.v))
        out = empty_rows(dev, q.size, bf16)
        with rows_of(dev, bf16):
            cache.attention(0, [(put_rows(dev, p.q, bf16), out, dr.Pass(dev.ctx, pos))], 4, sliding_window=12, scale=0.08)
        got[5, 1], got[9, 3] = True, True
        assert np.array_equal(np.isnan(dev.get(out.float())).reshape(got.shape), got)


def test_scale_signs_and_zero(dev):
    rng = np.random.default_rng(8)
    p = Problem(rng, 4, 2, 128, 200, range(150, 200))
    for scale in (-1 / math.sqrt(128), 0.0, 1e-3, 2 / math.sqrt(128)):
        run(dev, [p], scale=scale)
    p.q *= np.exp2(rng.integers(-40, 20, (50, 4, 1))).astype(np.float32)
    run(dev, [p], scale=1e-6)


def test_large_scale_needs_the_kernel_forced(dev):
    rng = np.random.default_rng(9)
    p = Problem(rng, 4, 2, 128, 100, range(90, 100))
    with pytest.raises(dr.DrError) as e:
        run(dev, [p], scale=1.0)
    assert e.value.status == dr.DR_ERR_UNSUPPORTED
    run(dev, [p], scale=1.0, kernel=dr.KERNEL_FP8)
    for kernel in (dr.KERNEL_STAGED, dr.KERNEL_STREAMS, dr.KERNEL_HILO):
        with pytest.raises(dr.DrError) as e:
            run(dev, [p], kernel=kernel)
        assert e.value.status == dr.DR_ERR_UNSUPPORTED


def test_forced_fp8_means_auto_elsewhere(dev):
    """The 8 bit family forced on a bf16 layer changes nothing, its scale limit
    included."""
    rng = np.random.default_rng(10)
    cache = dr.StepCache(dev.ctx, 64, [2], [128])
    p = dr.Pass(dev.ctx, range(64))
    x = dev.put(rng.standard_normal(64 * 256).astype(np.float32))
    cache.store(0, p, x, x)
    a, b = dev.empty(64 * 256), dev.empty(64 * 256)
    cache.attention(0, [(x, a, p)], 2, scale=0.05)
    dev.ctx.set_kernel(dr.KERNEL_FP8)
    try:
        cache.attention(0, [(x, b, p)], 2, scale=0.05)
        with pytest.raises(dr.DrError) as e:
            cache.attention(0, [(x, b, p)], 2, scale=1.0)
        assert e.value.status == dr.DR_ERR_UNSUPPORTED
    finally:
        dev.ctx.set_kernel(dr.KERNEL_AUTO)
    assert np.array_equal(dev.get(a), dev.get(b))


@pytest.mark.parametrize("q16,o16", [(True, False), (False, True)])
def test_mixed_row_types(dev, q16, o16):
    """bf16 Q with f32 output and the reverse."""
    rng = np.random.default_rng(11)
    for h, hkv, hd, n, pos in ((8, 2, 128, 200, range(150, 200)), (4, 2, 256, 90, [3]), (2, 1, 72, 90, range(30, 90))):
        p = Problem(rng, h, hkv, hd, n, pos)
        if q16:
            p.q = bf16_round(p.q)
        cache = dr.StepCache(dev.ctx, n, [hkv], [hd], precision=[dr.PRECISION_FP8])
        cache.store(0, dr.Pass(dev.ctx, range(n)), dev.put(p.k), dev.put(p.v))
        out = empty_rows(dev, p.q.size, o16)
        dev.ctx.set_q_dtype(dr.DTYPE_BF16 if q16 else dr.DTYPE_F32)
        dev.ctx.set_o_dtype(dr.DTYPE_BF16 if o16 else dr.DTYPE_F32)
        try:
            cache.attention(0, [(put_rows(dev, p.q, q16), out, dr.Pass(dev.ctx, pos))], h, scale=1 / math.sqrt(hd))
        finally:
            dev.ctx.set_q_dtype(dr.DTYPE_F32)
            dev.ctx.set_o_dtype(dr.DTYPE_F32)
        k, v = stored(p.k), stored(p.v)
        want, weighted = attend(p.q, k, v, p.pos, 1 / math.sqrt(hd))
        check(dev.get(out.float()), want, bound(p.q, k, v, weighted, want, 1 / math.sqrt(hd), o16))


def test_noalloc_gives_the_same_bits(dev):
    rng = np.random.default_rng(12)
    p = Problem(rng, 8, 2, 128, 900, [899])
    cache = dr.StepCache(dev.ctx, p.n, [p.hkv], [p.hd], precision=[dr.PRECISION_FP8])
    cache.store(0, dr.Pass(dev.ctx, range(p.n)), dev.put(p.k), dev.put(p.v))
    outs = [dev.empty(p.q.size) for _ in range(3)]
    q, ps = dev.put(p.q), dr.Pass(dev.ctx, p.pos)
    for i, o in enumerate(outs):
        cache.attention(0, [(q, o, ps)], p.h, scale=0.1, noalloc=i == 1)
    a, b, c = (dev.get(o) for o in outs)
    assert np.array_equal(a, b) and np.array_equal(a, c)


# ---- the step calls: store and attention together, with the whole epilogue


def epilogue64(x, kind, pos, w, bias, eps, table, rot, v_norm):
    """[n, heads, hd] rows through bias, norm and RoPE as the oracle does them."""
    n, heads, hd = x.shape
    x = x.reshape(n, heads * hd).copy()
    if bias is not None:
        x = x + bias[None]
    x = x.reshape(n, heads, hd).astype(np.float32)
    if kind == "v":
        if v_norm:
            s = np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True) + eps).astype(np.float32)
            x = x * (np.float32(1) / s)
        return x
    if w is not None:
        s = np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True) + eps).astype(np.float32)
        x = x * (np.float32(1) / s) * w
    if rot:
        half = rot // 2
        t = np.asarray(table).reshape(-1, half, 2)[pos][:, None]
        sn, cs = t[..., 0], t[..., 1]
        a, b = x[..., :half].copy(), x[..., half:rot].copy()
        x[..., :half], x[..., half:rot] = a * cs - b * sn, a * sn + b * cs
    return x


@pytest.mark.parametrize("h,hkv,hd,rot", [(4, 2, 64, 64), (4, 2, 128, 128), (6, 2, 128, 64), (4, 2, 256, 256),
                                          (2, 1, 512, 512), (4, 2, 512, 128), (3, 3, 80, 72), (4, 4, 128, 0)])
@pytest.mark.parametrize("pos", [range(70, 130), [0, 1, 31, 40, 90, 91, 92, 93, 129]], ids=["run", "list"])
@pytest.mark.parametrize("epi", ["", "b", "n", "bnv"])
def test_step_with_epilogue(dev, h, hkv, hd, rot, pos, epi):
    """dr_attention_step_rows on fused rows: what it leaves in the cache is the
    8 bit form of the epilogue's rows, and its attention reads that."""
    rng = np.random.default_rng(hd + rot + len(epi) + len(pos))
    n, pos, eps = 130, list(pos), 1e-6
    m = len(pos)
    fused = (h + 2 * hkv) * hd
    R = rng.standard_normal((m, fused)).astype(np.float32)
    K, V = (rng.standard_normal((n, hkv, hd)).astype(np.float32) for _ in range(2))
    kw, qn, kn, bq, bk, bv, table = {}, None, None, None, None, None, None
    if "n" in epi:
        qn, kn = (rng.uniform(0.5, 1.5, hd).astype(np.float32) for _ in range(2))
        kw.update(q_norm_w=dev.put(qn), k_norm_w=dev.put(kn))
    if "b" in epi:
        bq, bk, bv = ((0.1 * rng.standard_normal(c * hd)).astype(np.float32) for c in (h, hkv, hkv))
        kw.update(bq=dev.put(bq), bk=dev.put(bk), bv=dev.put(bv))
    if "v" in epi:
        kw.update(v_norm=True)
    if rot:
        table = orc.rope_table(n, rot, 10000.0)
        kw.update(rope=dr.Rope(dev.ctx, n, rot, 10000.0))
    cache = dr.StepCache(dev.ctx, n, [hkv], [hd], precision=[dr.PRECISION_FP8])
    cache.store(0, dr.Pass(dev.ctx, range(n)), dev.put(K), dev.put(V))
    p, rows, out = dr.Pass(dev.ctx, pos), dev.put(R), dev.empty(m * h * hd)
    base = rows.data_ptr()
    cache.step_rows(0, [(base, out, p, base + 4 * h * hd, base + 4 * (h + hkv) * hd)], h, fused, fused,
                    scale=1 / math.sqrt(hd), eps=eps, **kw)
    q = epilogue64(R[:, :h * hd].reshape(m, h, hd), "q", pos, qn, bq, eps, table, rot, False)
    k = epilogue64(R[:, h * hd:(h + hkv) * hd].reshape(m, hkv, hd), "k", pos, kn, bk, eps, table, rot, False)
    v = epilogue64(R[:, (h + hkv) * hd:].reshape(m, hkv, hd), "v", pos, None, bv, eps, table, rot, "v" in epi)
    gk, gv = dev.empty(m * hkv * hd), dev.empty(m * hkv * hd)
    cache.gather_pass(0, p, gk, gv)
    gk, gv = dev.get(gk).reshape(m, hkv, hd), dev.get(gv).reshape(m, hkv, hd)
    for got, x in ((gk, k), (gv, v)):
        # the epilogue's f32 roundings differ by a few 2^-23 of the row's size; a
        # value so close to the middle of two codes may take either: a whole step
        # (2^-3 of the value, or 2^-9 of the scale's unit), rarely
        want = stored(x)
        unit = np.exp2(np.ceil(np.log2(np.abs(x).max(-1, keepdims=True))) - 8)
        assert (np.abs(got - want) <= np.maximum(np.abs(want) / 8, unit * 2.0 ** -9) * 1.0001).all()
        assert (got != want).mean() < 1e-3 + 2.0 / want.size
    K, V = stored(K), stored(V)
    K[pos], V[pos] = gk, gv
    want, weighted = attend(q, K, V, pos, 1 / math.sqrt(hd))
    # (q after the epilogue: the kernel's f32 rounding against numpy's, 8 steps of 2^-24)
    tol = bound(q, K, V, weighted, want, 1 / math.sqrt(hd), False)
    size = np.abs(q).max() * np.abs(K).sum(-1).max() / math.sqrt(hd)
    check(dev.get(out), want, tol + weighted * 2 * size * 2.0 ** -21, "attention")


def test_step_is_store_and_attention(dev):
    """dr_attention_step, twice over a batch: the same bits as the two calls."""
    rng = np.random.default_rng(20)
    n, h, hkv, hd = 200, 8, 2, 128
    outs = []
    K, V = (rng.standard_normal((2, n, hkv, hd)).astype(np.float32) for _ in range(2))
    act = [list(range(150, 200)), [0, 3, 4, 5, 6, 7, 64, 199]]
    Q = [rng.standard_normal((len(a), h, hd)).astype(np.float32) for a in act]
    kn = dev.put(rng.uniform(0.5, 1.5, hd).astype(np.float32))
    for together in (True, False):
        cache = dr.StepCache(dev.ctx, n, [hkv], [hd], n_batch=2, precision=[dr.PRECISION_FP8])
        ps = [dr.Pass(dev.ctx, a) for a in act]
        o = [dev.empty(q.size) for q in Q]
        for b in range(2):
            cache.store(0, dr.Pass(dev.ctx, range(n)), dev.put(K[b]), dev.put(V[b]), batch=b)
        new = [(dev.put(K[b][act[b]] * 2), dev.put(V[b][act[b]] - 1)) for b in range(2)]
        if together:
            cache.step(0, [(dev.put(Q[b]), o[b], ps[b], *new[b]) for b in range(2)], h, scale=0.08, q_norm_w=kn,
                       k_norm_w=kn)
        else:
            for b in range(2):
                cache.store(0, ps[b], *new[b], k_norm_w=kn, batch=b)
            cache.attention(0, [(dev.put(Q[b]), o[b], ps[b]) for b in range(2)], h, scale=0.08, q_norm_w=kn)
        outs.append([dev.get(x) for x in o])
    assert all(np.array_equal(a, b) for a, b in zip(*outs))


def test_captured_step_replays(dev):
    """A step in a hipGraph: several replays, with eager work between them and new
    rows in the same buffers, each equal to the eager call."""
    t = dev.t
    rng = np.random.default_rng(21)
    n, h, hkv, hd = 300, 8, 2, 128
    cache = dr.StepCache(dev.ctx, n, [hkv], [hd], precision=[dr.PRECISION_FP8])
    K = rng.standard_normal((n, hkv, hd)).astype(np.float32)
    cache.store(0, dr.Pass(dev.ctx, range(n)), dev.put(K), dev.put(K))
    p = dr.Pass(dev.ctx, range(290, 300))
    q, k, v = (dev.put(rng.standard_normal(10 * c * hd).astype(np.float32)) for c in (h, hkv, hkv))
    out, eager = dev.empty(10 * h * hd), dev.empty(10 * h * hd)
    gk, gv = dev.empty(10 * hkv * hd), dev.empty(10 * hkv * hd)
    cache.step(0, [(q, out, p, k, v)], h, scale=0.08)
    dev.stream.synchronize()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph, stream=dev.stream):
        cache.step(0, [(q, out, p, k, v)], h, scale=0.08)
        cache.gather_pass(0, p, gk, gv)
    for i in range(4):
        with t.cuda.stream(dev.stream):
            for x in (q, k, v):
                x.copy_(t.randn_like(x))
            out.fill_(float("nan"))
            gk.fill_(float("nan"))
            graph.replay()
        got, got_k = dev.get(out), dev.get(gk)
        cache.step(0, [(q, eager, p, k, v)], h, scale=0.08)
        assert np.array_equal(got, dev.get(eager)), i
        assert np.array_equal(got_k.reshape(-1, hkv, hd), stored(dev.get(k).reshape(-1, hkv, hd)).astype(np.float32)), i


def test_split_pass_and_other_streams(dev):
    """The passes that dr_cache_split_active_dev fills drive store, attention and
    read back, with the context moved to another stream in between."""
    t = dev.t
    rng = np.random.default_rng(22)
    n, h, hkv, hd = 257, 4, 2, 128
    cache = dr.StepCache(dev.ctx, n, [hkv], [hd], precision=[dr.PRECISION_FP8])
    K, V = (rng.standard_normal((n, hkv, hd)).astype(np.float32) for _ in range(2))
    cache.store(0, dr.Pass(dev.ctx, range(n)), dev.put(K), dev.put(V))
    seq = rng.integers(5, 999, n).astype(np.int32)
    cache.update_seq_dev(dev.put(seq))
    mask = np.zeros(n, np.uint8)
    mask[rng.permutation(n)[:41]] = 1
    act, rest = dr.Pass(dev.ctx, []), dr.Pass(dev.ctx, [])
    na, nc = cache.split_active_dev(dev.put(seq), dev.put(mask), n, 5, act, rest)
    pos = act.positions()
    q, k, v = (rng.standard_normal((na, c, hd)).astype(np.float32) for c in (h, hkv, hkv))
    dq, dk, dv = dev.put(q), dev.put(k), dev.put(v)
    out, gk, gv = dev.empty(q.size), dev.empty(nc * hkv * hd), dev.empty(nc * hkv * hd)
    dev.stream.synchronize()
    other = t.cuda.Stream()
    dev.ctx.set_stream(other.cuda_stream)
    try:
        cache.store(0, act, dk, dv)
        dev.ctx.set_stream(dev.stream.cuda_stream)
        cache.attention(0, [(dq, out, act)], h, scale=0.09)
        dev.ctx.set_stream(other.cuda_stream)
        cache.gather_pass(0, rest, gk, gv)
        other.synchronize()
    finally:
        dev.ctx.set_stream(dev.stream.cuda_stream)
    K2, V2 = stored(K), stored(V)
    left = rest.positions()
    assert np.array_equal(dev.get(gk).reshape(nc, hkv, hd), K2[left].astype(np.float32))
    assert np.array_equal(dev.get(gv).reshape(nc, hkv, hd), V2[left].astype(np.float32))
    K2[pos], V2[pos] = stored(k), stored(v)
    want, weighted = attend(q, K2, V2, pos, 0.09)
    check(dev.get(out), want, bound(q, K2, V2, weighted, want, 0.09, False))


def test_long_cache_past_32_bit_offsets(dev):
    """Keys past 4 GB of a plane: the last KV head of 33, window around the end."""
    n, hkv, hd = 1 << 20, 33, 128
    rng = np.random.default_rng(23)
    cache = dr.StepCache(dev.ctx, n, [hkv], [hd], precision=[dr.PRECISION_FP8])
    tail = 100
    K, V = (rng.standard_normal((tail, hkv, hd)).astype(np.float32) for _ in range(2))
    cache.store(0, dr.Pass(dev.ctx, range(n - tail, n)), dev.put(K), dev.put(V))
    for pos in ([n - 1], range(n - 20, n)):
        q = rng.standard_normal((len(pos), hkv, hd)).astype(np.float32)
        out = dev.empty(q.size)
        cache.attention(0, [(dev.put(q), out, dr.Pass(dev.ctx, pos))], hkv, sliding_window=70, scale=0.09)
        k, v = stored(K), stored(V)
        want, weighted = attend(q, k, v, [p - (n - tail) for p in pos], 0.09, 70)
        check(dev.get(out), want, bound(q, k, v, weighted, want, 0.09, False))
