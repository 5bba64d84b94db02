"""What holding K and V in 8 bits costs against the rows that were stored (CPU
only, in float64 but for the rounding to codes): the size that the library's
header states for DR_PRECISION_FP8 layers."""
from __future__ import annotations

import math

import numpy as np
import pytest

from fp8_reference import attend, stored
from helpers import bf16_round


@pytest.mark.parametrize("h,hkv,hd,keys,rows", [(2, 2, 128, 768, 256), (4, 1, 64, 517, 100), (2, 1, 256, 2553, 32)])
def test_error_against_the_stored_rows(h, hkv, hd, keys, rows):
    """e4m3 keeps 4 bits: a value in [1, 2) is off by a uniform +-2^-4, 2^-4 /
    sqrt(3) = 3.6 % rms, and by 3.6 % / 2 at the upper end of its binade: 2.5 % of
    values spread over it.  N(0, 1) rows at 1 / sqrt(head_dim): scores are off by
    2.5 % and values too, outputs by 2.5 % * sqrt(2) = 3.6 % rms, 2.8 % mean-abs of
    their rms size; between 2.3 and 4 % is asked.  Twice the scale doubles the
    scores' part; bf16, with 8 bits, is 2^4 below."""
    rng = np.random.default_rng(hd)
    q, k, v = (rng.standard_normal((n, c, hd)).astype(np.float32) for n, c in ((rows, h), (keys, hkv), (keys, hkv)))

    def off(scale, k2, v2):
        want = attend(q, k, v, [0] * rows, scale)[0]
        e = np.abs(attend(q, k2, v2, [0] * rows, scale)[0] - want)
        return e.mean() / math.sqrt((want ** 2).mean()), e.max()

    scale = 1 / math.sqrt(hd)
    mean, most = off(scale, stored(k), stored(v))
    assert 0.023 < mean < 0.04 and most < 0.04
    assert mean < off(2 * scale, stored(k), stored(v))[0] < 3 * mean
    assert 8 * off(scale, bf16_round(k), bf16_round(v))[0] < mean
