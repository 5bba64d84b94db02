"""Calls whose passes are all empty do nothing and succeed, on layers of every
precision, also with a whole epilogue.  Needs an MI355X."""
from __future__ import annotations

import numpy as np
import pytest

import dr_attn as dr

from test_gpu_parity import dev, say, torch  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("precision", [dr.PRECISION_BF16, dr.PRECISION_HILO, dr.PRECISION_FP8])
@pytest.mark.parametrize("h,hkv,hd", [(4, 2, 128), (4, 4, 64), (2, 1, 512)])
@pytest.mark.parametrize("slots", [1, 2])
def test_empty_passes(dev, precision, h, hkv, hd, slots):
    n = 300
    cache = dr.StepCache(dev.ctx, n, [hkv], [hd], n_batch=slots, precision=[precision])
    rng = np.random.default_rng(hd)
    k = dev.put(rng.standard_normal((n, hkv, hd)).astype(np.float32))
    for b in range(slots):
        cache.store(0, dr.Pass(dev.ctx, range(n)), k, k, batch=b)
    held = dev.empty(n * hkv * hd)
    cache.gather_pass(0, dr.Pass(dev.ctx, range(n)), held, dev.empty(n * hkv * hd))
    none = dr.Pass(dev.ctx, [])
    w, q, out = dev.put(np.ones(hd, np.float32)), dev.put(np.zeros(h * hd, np.float32)), dev.empty(h * hd)
    epi = dict(q_norm_w=w, k_norm_w=w, v_norm=True, rope=dr.Rope(dev.ctx, n, hd, 1e4))
    for kv in (q, None):
        for kw in ({}, {"sliding_window": 7}, {"causal_prefix": 9}):
            cache.attention(0, [(q, out, none)] * slots, h, scale=0.05, **kw)
            cache.attention(0, [(q, out, none)] * slots, h, scale=0.05, noalloc=True, **kw)
            cache.step(0, [(q, out, none, kv, kv)] * slots, h, scale=0.05, **kw)
            cache.step_epi(0, [(q, out, none, kv, kv)] * slots, h, scale=0.05, **kw, **epi)
            cache.step_rows(0, [(q, out, none, kv, kv)] * slots, h, h * hd, 0, scale=0.05, **kw)
    cache.store(0, none, None, None)
    cache.gather_pass(0, none, None, None)
    assert np.isnan(dev.get(out)).all()  # (never written)
    after = dev.empty(n * hkv * hd)
    cache.gather_pass(0, dr.Pass(dev.ctx, range(n)), after, dev.empty(n * hkv * hd))
    assert np.array_equal(dev.get(held), dev.get(after))
