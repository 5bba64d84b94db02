"""Calls on DR_PRECISION_FP8 layers that could overlap on the device, and what
keeps them apart: a context that switches streams between split calls, two
contexts on two streams that share the GPU's fixed scratch, two host threads on
one context, captured graphs that share a context's workspace, among them calls
on the slow way of scales far apart.  Every output equals that of the same call
made alone, bit for bit.  Needs an MI355X."""
from __future__ import annotations

import math
import threading

import numpy as np
import pytest

import dr_attn as dr

from test_gpu_concurrency import _empty, say, torch_mod  # noqa: F401

pytestmark = pytest.mark.gpu

# (query heads, KV heads, head dim, cached, active, key splits, rows a wave, spread of the scales)
SHAPES = {
    "rows": (8, 2, 128, 1500, 40, 5, 0, 0),
    "one": (16, 4, 128, 3000, 1, 0, 0, 0),
    "wide": (4, 2, 512, 700, 40, 3, 32, 0),
    "far": (4, 2, 256, 700, 40, 4, 0, 30),
    "wide_far": (4, 2, 512, 500, 70, 2, 32, 30),
}


def problem(torch, ctx, stream, name):
    h, hkv, hd, n_p, n_c, split, rows, spread = SHAPES[name]
    rng = np.random.default_rng(sum(map(ord, name)))
    n = n_p + n_c
    cache = dr.StepCache(ctx, n, [hkv], [hd], precision=[dr.PRECISION_FP8])
    K, V = (rng.standard_normal((n, hkv, hd)).astype(np.float32) for _ in range(2))
    V *= np.exp2(rng.integers(-spread, spread + 1, (n, hkv, 1))).astype(np.float32)
    with torch.cuda.stream(stream):
        K, V = torch.from_numpy(K).cuda(), torch.from_numpy(V).cuda()
        Qs = [torch.from_numpy(rng.standard_normal(n_c * h * hd).astype(np.float32)).cuda() for _ in range(3)]
    cache.store(0, dr.Pass(ctx, range(n)), K, V)
    stream.synchronize()
    p = dr.Pass(ctx, range(n_p, n))

    def call(q, o, noalloc=False):
        cache.attention(0, [(q, o, p)], h, scale=1 / math.sqrt(hd), noalloc=noalloc)

    ctx.set_split(split)
    ctx.set_wave_rows(rows)
    size, want = n_c * h * hd, []
    for q in Qs:
        o = _empty(torch, stream, size)
        call(q, o)
        stream.synchronize()
        want.append(o.cpu().numpy())
    info = ctx.last_launch()
    assert info["kernel"] == dr.KERNEL_FP8 and info["n_split"] > 1
    assert np.isfinite(want[0]).all()
    say(f"{name}: {info}")
    return call, Qs, size, want


@pytest.mark.parametrize("name", list(SHAPES))
def test_stream_switch_orders_the_contexts_work(torch_mod, name):
    torch = torch_mod
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    ctx = dr.Context(0)
    ctx.set_stream(sa.cuda_stream)
    try:
        call, Qs, size, want = problem(torch, ctx, sa, name)
        for rep in range(3):
            outs = []
            for i, q in enumerate(Qs):
                s = (sa, sb)[(i + rep) % 2]
                ctx.set_stream(s.cuda_stream)
                o = _empty(torch, s, size)
                call(q, o)
                outs.append(o)
            (sa, sb)[(len(Qs) - 1 + rep) % 2].synchronize()
            for i, o in enumerate(outs):
                assert np.array_equal(o.cpu().numpy(), want[i]), (rep, i)
    finally:
        ctx.set_stream(0)


@pytest.mark.parametrize("pair", [("rows", "wide"), ("one", "far"), ("wide_far", "rows")], ids="-".join)
def test_noalloc_calls_on_two_streams_take_turns(torch_mod, pair):
    torch = torch_mod
    streams = [torch.cuda.Stream() for _ in pair]
    ctxs = [dr.Context(0) for _ in pair]
    for c, s in zip(ctxs, streams):
        c.set_stream(s.cuda_stream)
    probs = [problem(torch, c, s, name) for c, s, name in zip(ctxs, streams, pair)]
    outs = {}
    for rep in range(4):
        for i in range(3):
            for k, (s, (call, Qs, size, _)) in enumerate(zip(streams, probs)):
                o = _empty(torch, s, size)
                call(Qs[i], o, noalloc=True)
                outs[rep, i, k] = o
    for s in streams:
        s.synchronize()
    for (rep, i, k), o in outs.items():
        assert np.array_equal(o.cpu().numpy(), probs[k][3][i]), (rep, i, k)


@pytest.mark.parametrize("name", ["rows", "wide"])
def test_two_threads_on_one_context(torch_mod, name):
    torch = torch_mod
    st = torch.cuda.Stream()
    ctx = dr.Context(0)
    ctx.set_stream(st.cuda_stream)
    call, Qs, size, want = problem(torch, ctx, st, name)
    outs = [[_empty(torch, st, size) for _ in range(20)] for _ in range(2)]
    done, busy, errors = [[False] * 20 for _ in range(2)], [0, 0], []

    def run(t):
        try:
            for i in range(20):
                try:
                    call(Qs[0], outs[t][i])
                    done[t][i] = True
                except dr.DrError as e:
                    if e.status != dr.DR_ERR_BUSY:
                        raise
                    busy[t] += 1
        except Exception as e:  # reported below
            errors.append(repr(e))

    th = [threading.Thread(target=run, args=(t,)) for t in range(2)]
    for t in th:
        t.start()
    for t in th:
        t.join()
    st.synchronize()
    assert not errors, errors
    for t in range(2):
        for i in range(20):
            if done[t][i]:
                assert np.array_equal(outs[t][i].cpu().numpy(), want[0]), (t, i)
    assert sum(map(sum, done)) + sum(busy) == 40


@pytest.mark.parametrize("name", ["rows", "one", "wide", "far"])
def test_two_graphs_share_a_workspace(torch_mod, name):
    """Two captured calls of one context, replayed in turn with eager calls
    between them: the same tickets and split workspace, ready each time."""
    torch = torch_mod
    st = torch.cuda.Stream()
    ctx = dr.Context(0)
    ctx.set_stream(st.cuda_stream)
    call, Qs, size, want = problem(torch, ctx, st, name)
    outs, graphs = [_empty(torch, st, size) for _ in range(2)], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            call(Qs[i], outs[i])
        graphs.append(g)
    eager = _empty(torch, st, size)
    for rep in range(4):
        with torch.cuda.stream(st):
            for i in (0, 1):
                outs[i].fill_(float("nan"))
            graphs[rep % 2].replay()
            graphs[1 - rep % 2].replay()
        call(Qs[2], eager)
        st.synchronize()
        for i in (0, 1):
            assert np.array_equal(outs[i].cpu().numpy(), want[i]), (rep, i)
        assert np.array_equal(eager.cpu().numpy(), want[2])
