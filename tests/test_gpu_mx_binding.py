"""Codes that torch's arithmetic left in wider whole numbers, and strided ones, give the
products of the bytes that they stand for.  Needs an MI355X."""
from __future__ import annotations

import numpy as np
import pytest

import dr_attn as dr
from test_gpu_mx_matmul import acts, weights
from test_gpu_mx_rows import FILL, empty_rows, get_rows, put_rows
from test_gpu_parity import dev, torch  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", ["int64", "int32", "strided"])
@pytest.mark.parametrize("n", [1, 40])
def test_codes_of_other_tensors(dev, how, n):
    t = dev.t
    rng = np.random.default_rng(n)
    rows, cols = 64, 544
    w, up, a = weights(rng, rows, cols), weights(rng, rows, cols), acts(rng, n, cols, dr.MX_E2M1)

    def other(codes, scales):
        with t.cuda.stream(dev.stream):
            if how == "strided":
                wide = t.full((codes.shape[0], codes.shape[1] + 48), FILL, dtype=t.uint8, device="cuda")
                wide[:, 16:-32] = t.from_numpy(codes).cuda()
                return dr.MxRows(wide[:, 16:-32], t.from_numpy(scales).cuda(), dr.MX_E2M1)
            kind = getattr(t, how)
            return dr.MxRows(t.from_numpy(codes).cuda().to(kind), t.from_numpy(scales).cuda().to(kind), dr.MX_E2M1)

    results = []
    for make in (lambda r: put_rows(dev, *r, dr.MX_E2M1), lambda r: other(*r)):
        dw, dup, da = make(w), make(up), make(a)
        out, mid, back = dev.empty(n * rows), empty_rows(dev, n, rows, dr.MX_E4M3), dev.empty(n * cols)
        dr.mx_matmul(dev.ctx, dw, rows, cols, da, n, out)
        dr.mx_gated(dev.ctx, dw, dup, rows, cols, da, n, mid)
        dr.mx_dequantize(dev.ctx, da, n, cols, back)
        results.append([dev.get(out).copy(), *get_rows(dev, mid, n, rows), dev.get(back).copy()])
    assert np.abs(results[0][0]).max() > 0
    for x, y in zip(*results):
        assert np.array_equal(x, y)
