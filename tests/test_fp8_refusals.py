"""The 8 bit cache layers' refusals that need no GPU, and the format's reference
itself (CPU only)."""
from __future__ import annotations

import numpy as np

import dr_attn as dr
from fp8_reference import attend, e4m3_round, stored
from helpers import RowsSpec, Shape, brute_force


def test_null_arguments():
    lib = dr.load()
    assert lib.dr_cache_gather_pass(None, 0, 0, None, None, None) == dr.DR_ERR_INVALID
    assert "cache" in lib.dr_last_error().decode()
    assert lib.dr_cache_set_precision(None, 0, dr.PRECISION_FP8) == dr.DR_ERR_INVALID
    assert lib.dr_ctx_set_kernel(None, dr.KERNEL_FP8) == dr.DR_ERR_INVALID


def test_bad_precision_before_any_device():
    import ctypes

    lib = dr.load()
    one = (ctypes.c_size_t * 1)(1)
    h = ctypes.c_void_p()
    for bad in (-1, 3, 7):
        p = np.array([bad], np.int32)
        assert lib.dr_cache_create_layers(None, 1, 1, one, one, p.ctypes.data, 1, ctypes.byref(h)) == dr.DR_ERR_INVALID
        assert "precision" in lib.dr_last_error().decode()


def test_reference_codes():
    """e4m3_round against the list of e4m3 values."""
    codes = np.array(sorted({s * v for s in (1, -1) for v in
                             [m / 512 for m in range(8)] +
                             [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8) if (1 + m / 8) * 2.0 ** e <= 448]}))
    assert len(codes) == 253
    assert np.array_equal(e4m3_round(codes), codes)
    y = np.random.default_rng(0).uniform(-448, 448, 2000)
    y = np.concatenate([y, y * 2.0 ** -6, y * 2.0 ** -14])
    got = e4m3_round(y)
    assert np.isin(got, codes).all()
    assert np.allclose(np.abs(got - y), np.abs(codes[None] - y[:, None]).min(1), rtol=0, atol=0)


def test_reference_against_torch():
    import torch

    rng = np.random.default_rng(1)
    x = (rng.standard_normal((500, 64)) * np.exp2(rng.integers(-40, 40, (500, 1)))).astype(np.float32)
    m, e = torch.frexp(torch.from_numpy(x).abs().amax(-1, keepdim=True))
    e = torch.clamp(e - 9 + (m > 0.875).to(torch.int32), min=-126)
    want = torch.ldexp(torch.ldexp(torch.from_numpy(x), -e).to(torch.float8_e4m3fn).float(), e)
    assert np.array_equal(stored(x).astype(np.float32), want.numpy())


def test_reference_attention():
    rng = np.random.default_rng(2)
    n, h, hkv, hd, pos = 40, 4, 2, 8, [3, 9, 20, 39]
    q, k, v = rng.standard_normal((4, h, hd)), rng.standard_normal((n, hkv, hd)), rng.standard_normal((n, hkv, hd))
    for w, pre in ((None, None), (5, None), (None, 21), (7, 15), (0, None)):
        s = Shape(4, n, h, hkv, hd, sliding_window=w, causal_prefix=pre, scale=0.3)
        want = brute_force(q.reshape(-1), k.reshape(-1), v.reshape(-1), s, RowsSpec(pos), RowsSpec(range(n)))
        got = attend(q, k, v, pos, 0.3, w, pre)[0].reshape(4, -1)
        assert np.allclose(got, want, rtol=1e-12, atol=1e-13, equal_nan=True)
