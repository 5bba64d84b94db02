"""The products' tiles read nothing behind a plane of scale rows (CPU only): the
result cannot show it, as what is read there is not used."""
from __future__ import annotations

import pytest

import dr_attn as dr


@pytest.mark.parametrize("cols", [32, 96, 416, 512, 544, 576, 640, 672, 1056, 1120, 1184, 2336, 2880, 3584, 8224, 12320, 1 << 22])
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 255, 256, 257, 1024, 4099])
def test_scale_reads_end_with_the_plane(rows, cols):
    rows = min(rows, 2) if cols == 1 << 22 else rows
    assert dr.mx_scale_end(rows, cols) == rows * dr.mx_pitch(cols)  # all of it, and no more


def test_refusals():
    for rows, cols in ((0, 32), (1, 0), (1, 31), (1 << 40, 32)):
        with pytest.raises(dr.DrError):
            dr.mx_scale_end(rows, cols)
