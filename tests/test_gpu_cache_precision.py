"""dr_cache_set_precision while a stream is captured into a graph: a call that
changes nothing does nothing, one that would make or free planes is refused and
leaves the capture and the layer as they were.  Needs an MI355X."""
from __future__ import annotations

import math

import numpy as np
import pytest

import dr_attn as dr

from test_gpu_parity import say, torch  # noqa: F401

pytestmark = pytest.mark.gpu

KINDS = [dr.PRECISION_BF16, dr.PRECISION_HILO, dr.PRECISION_FP8]


def captured_step(torch, ctx, stream, kind, inside):
    """A captured attention call on a layer of `kind`, `inside(cache)` called within
    the capture; its output after two replays and the eager call's."""
    rng = np.random.default_rng(kind)
    n, h, hkv, hd, m = 70, 4, 2, 128, 20
    cache = dr.StepCache(ctx, n, [hkv], [hd], precision=[kind])
    with torch.cuda.stream(stream):
        K, V = (torch.from_numpy(rng.standard_normal((n, hkv, hd)).astype(np.float32)).cuda() for _ in range(2))
        q = torch.from_numpy(rng.standard_normal((m, h, hd)).astype(np.float32)).cuda()
        out, eager = torch.zeros_like(q), torch.zeros_like(q)
    p = dr.Pass(ctx, range(n - m, n))
    cache.store(0, dr.Pass(ctx, range(n)), K, V)
    cache.attention(0, [(q, eager, p)], h, scale=1 / math.sqrt(hd))
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        inside(cache)
        cache.attention(0, [(q, out, p)], h, scale=1 / math.sqrt(hd))
    for _ in range(2):
        with torch.cuda.stream(stream):
            out.fill_(float("nan"))
            graph.replay()
        stream.synchronize()
        assert np.array_equal(out.cpu().numpy(), eager.cpu().numpy())
    return cache


@pytest.fixture(params=["own", "torch"])
def ctx_stream(request, torch):
    """A context on the stream that it makes itself, or on one of torch's."""
    ctx = dr.Context(0)
    if request.param == "own":
        return ctx, torch.cuda.ExternalStream(ctx.stream)
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    return ctx, stream


@pytest.mark.parametrize("kind", KINDS)
def test_the_same_precision_again(torch, ctx_stream, kind):
    captured_step(torch, *ctx_stream, kind, lambda cache: cache.set_precision(0, kind))


@pytest.mark.parametrize("kind", KINDS)
def test_a_change_under_capture_is_refused(torch, ctx_stream, kind):
    def change(cache):
        for other in KINDS:
            if other != kind:
                with pytest.raises(dr.DrError) as e:
                    cache.set_precision(0, other)
                assert e.value.status == dr.DR_ERR_INVALID and "capture" in str(e.value)

    cache = captured_step(torch, *ctx_stream, kind, change)
    for other in KINDS:
        cache.set_precision(0, other)  # (free to change once no stream is captured)
