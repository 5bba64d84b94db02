"""What the binding's MxRows takes for codes and scales (CPU only)."""
from __future__ import annotations

import types

import pytest
import torch

import dr_attn as dr


class OnGpu:
    """A CPU tensor that says it is on a GPU: its address is held, never read."""

    def __init__(self, t):
        self.t = t
        self.is_cuda = True

    def __getattr__(self, name):
        return getattr(self.t, name)

    def __lt__(self, x):
        return self.t < x

    def __gt__(self, x):
        return self.t > x


CODES = torch.arange(4 * 16).reshape(4, 16) * 4 % 256
SCALES = torch.full((4, 4), 127)


def test_bytes_are_used_in_place():
    for t in (torch.uint8, torch.int8):
        codes, scales = OnGpu(CODES.to(t)), OnGpu(SCALES.to(torch.uint8))
        r = dr.MxRows(codes, scales, dr.MX_E2M1)
        assert (r.c.codes, r.c.scales) == (codes.data_ptr(), scales.data_ptr()) and not r.copied
        assert r.written() is r.c
    f8 = OnGpu(torch.ones(4, 32).to(torch.float8_e4m3fn))
    assert dr.MxRows(f8, OnGpu(SCALES.byte()), dr.MX_E4M3).c.codes == f8.data_ptr()
    assert dr.MxRows(4096, 8192, dr.MX_E4M3).c.codes == 4096  # an address is taken as it is


@pytest.mark.parametrize("t", [torch.int64, torch.int32, torch.int16])
def test_wider_whole_numbers_become_bytes(t):
    r = dr.MxRows(OnGpu(CODES.to(t)), OnGpu(SCALES.to(t)), dr.MX_E2M1)
    assert r.codes.dtype == r.scales.dtype == torch.uint8 and r.codes.is_contiguous()
    assert torch.equal(r.codes, CODES.byte()) and torch.equal(r.scales, SCALES.byte())
    assert (r.c.codes, r.c.scales) == (r.codes.data_ptr(), r.scales.data_ptr())


def test_strided_bytes_become_contiguous():
    wide = torch.arange(128, dtype=torch.uint8).reshape(4, 32)
    r = dr.MxRows(OnGpu(wide[:, 8:24]), OnGpu(SCALES.byte()), dr.MX_E2M1)
    assert r.codes.is_contiguous() and torch.equal(r.codes, wide[:, 8:24]) and r.c.codes == r.codes.data_ptr()
    turned = OnGpu(SCALES.byte()[:, :1].expand(4, 4))
    assert dr.MxRows(OnGpu(CODES.byte()), turned, dr.MX_E2M1).copied


def test_copies_are_not_written():
    """A result in the copy would never reach the given tensor."""
    r = dr.MxRows(OnGpu(CODES), OnGpu(SCALES.byte()), dr.MX_E2M1)
    ctx = types.SimpleNamespace(h=None, lib=dr.load())
    calls = [lambda: dr.mx_quantize(ctx, 4096, 4, 32, r), lambda: dr.rms_norm_mx(ctx, 4096, 4, 32, r),
             lambda: dr.mx_gated(ctx, r, r, 32, 32, r, 4, r)]
    for call in calls:
        with pytest.raises(TypeError, match="cannot be written"):
            call()


@pytest.mark.parametrize("codes,error,word", [
    (OnGpu(torch.zeros(4, 16)), TypeError, "codes"), (OnGpu(torch.zeros(4, 16, dtype=torch.bfloat16)), TypeError, "codes"),
    (OnGpu(torch.full((4, 16), 256)), ValueError, "codes"), (OnGpu(torch.full((4, 16), -1)), ValueError, "codes"),
    (torch.zeros(4, 16, dtype=torch.uint8), TypeError, "GPU")])
def test_refusals(codes, error, word):
    with pytest.raises(error, match=word):
        dr.MxRows(codes, OnGpu(SCALES.byte()), dr.MX_E2M1)
    with pytest.raises(error):
        dr.MxRows(OnGpu(CODES.byte()), codes, dr.MX_E2M1)
