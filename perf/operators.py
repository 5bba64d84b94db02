"""The 8 bit KV cache: writing rows into it, reading them back, and the attention
that reads it, over the shapes a denoise loop calls them at.

Kinds of case (a case is a dict of plain values; head counts, head dims and
lengths are those of tests/helpers.py, bench.py and perf/cases.py):

  store   K and V rows quantised into a cache layer, then read back as the f32
          values that the layer now stands for.  "run": consecutive positions
          (a canvas, a prompt), read back at the same positions; "list": the
          scattered positions of a late denoise step, every position read back.
  attend  one layer's attention of the active rows over all cached positions;
          "run" are the last rows of the sequence, "list" scattered ones.
          io "f32": f32 rows in and out, "bf16": bf16 rows in and out.
  step    both in one call, as a denoise step's layer makes it: the active rows
          are stored and then attend; the stored rows are read back as well.

The format: head_dim values of one position of one KV head share a power of two
2^e, the smallest that keeps the largest of them within e4m3's 448; each value is
x / 2^e rounded to e4m3 (nearest, ties to even).
"""
from __future__ import annotations

import math
import pathlib
import sys

import numpy as np
import torch

own = False

# name: (query heads, KV heads, head dim)
MODELS = {
    "llada": (32, 32, 128),
    "dream": (28, 4, 128),
    "llada_moe": (16, 16, 128),
    "gqa": (32, 8, 128),
    "gemma_sliding": (16, 8, 256),
    "gemma_global": (16, 2, 512),
    "small": (8, 2, 64),
    "odd": (6, 3, 80),
}


def _case(op, model, keys, rows, layout="run", batch=1, io="f32", window=0, prefix=0):
    """window 0: none; prefix 0: none (rows below it are causal)."""
    return {"op": op, "model": model, "keys": keys, "rows": rows, "layout": layout, "batch": batch, "io": io,
            "window": window, "prefix": prefix}


# ------------------------------------------------------------------ cases


def listed():
    return [
        # one fresh position of a small grouped-head layer: latency alone
        dict(_case("store", "dream", 769, 1), name="store_one"),
        # the canvas rows of LLaDA-8B's denoise step
        dict(_case("store", "llada", 768, 256), name="store_canvas"),
        # a late step: the still masked and just changed positions, anywhere in the sequence
        dict(_case("store", "llada_moe", 2553, 181, layout="list"), name="store_list"),
        # the first pass of a long prompt
        dict(_case("store", "gqa", 32768, 32768), name="store_prompt"),
        # a single position asks, bf16 rows, a cache of ordinary length
        dict(_case("attend", "gqa", 4097, 1, io="bf16"), name="attend_one"),
        # the same over a very long cache, f32 rows
        dict(_case("attend", "gqa", 131072, 1), name="attend_one_long"),
        # LLaDA-8B's denoise step: 256 canvas rows over 512 + 256 positions
        dict(_case("attend", "llada", 768, 256), name="attend_canvas"),
        # guidance pair of a late step, scattered rows, ragged length
        dict(_case("attend", "dream", 1321, 181, layout="list", batch=2), name="attend_list"),
        # the sliding-window layers at head dim 256, bf16 rows
        dict(_case("attend", "gemma_sliding", 4352, 256, io="bf16", window=1024), name="attend_window"),
        # the global layers at head dim 512
        dict(_case("attend", "gemma_global", 4352, 256), name="attend_global"),
        # a first pass: every position asks, the prompt's rows causally, bf16 rows
        dict(_case("attend", "llada", 4096, 4096, io="bf16", prefix=3840), name="attend_first"),
        # a layer of a denoise step: 512 rows stored and attending over 2041 + 512
        dict(_case("step", "llada_moe", 2553, 512), name="step_canvas"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {n: max(work(c)[n] for c in listed()) for n in ("bytes", "flops")}
    while True:
        c = _draw(rng)
        w = work(c)
        pairs = MODELS[c["model"]][0] * c["rows"] * c["keys"] * c["batch"]
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and (c["op"] == "store" or pairs <= 1 << 29):
            return c


def _draw(rng):
    op = rng.choice(["store", "attend", "attend", "attend", "step"])
    model = rng.choice(list(MODELS))
    keys = _log(rng, 1, 131072 if op == "attend" and rng.random() < 0.5 else 16384)
    rows = min(keys, rng.choice([1, _log(rng, 1, 64), _log(rng, 16, 4096)]))
    layout = rng.choice(["run", "list"])
    batch = rng.choice([1, 1, 2, 3])
    if op == "store":
        return _case(op, model, keys, rows, layout, batch)
    window = rng.choice([0, 0, _log(rng, 1, 2048)])
    prefix = rng.choice([0, 0, rng.randint(0, keys)])
    return _case(op, model, keys, rows, layout, batch, rng.choice(["f32", "bf16"]), window, prefix)


def _positions(case, rng):
    """The active positions of one batch slot, ascending."""
    if case["layout"] == "run":
        return np.arange(case["keys"] - case["rows"], case["keys"])
    return np.sort(rng.permutation(case["keys"])[: case["rows"]])


def _band(case, pos):
    """[lo, hi) of the positions that each query position sees."""
    n, w, pre = case["keys"], case["window"], case["prefix"]
    lo = np.maximum(0, pos - w + 1) if w else np.zeros_like(pos)
    hi = np.minimum(n, pos + w) if w else np.full_like(pos, n)
    return lo, np.where(pos < pre, np.minimum(hi, pos + 1), hi)


def work(case):
    h, hkv, hd = MODELS[case["model"]]
    n, rows, batch = case["keys"], case["rows"], case["batch"]
    kv8 = 2 * hkv * (hd + 1)  # a position's K and V in 8 bits, with their scales
    kv32 = 8 * hkv * hd  # the same in f32
    back = n if case["op"] == "store" and case["layout"] == "list" else rows
    b = batch * (rows * (kv32 + kv8) + back * (kv8 + kv32)) if case["op"] != "attend" else 0
    if case["op"] == "store":
        return {"bytes": b, "flops": 0}
    pos = _positions(case, np.random.default_rng(0))
    lo, hi = _band(case, pos)
    seen = np.zeros(n + 1, np.int64)
    np.add.at(seen, lo, 1)
    np.add.at(seen, hi, -1)
    keys = int((np.cumsum(seen)[:n] > 0).sum())
    if case["op"] == "step":  # the rows just stored need not come from memory again
        keys = max(0, keys - rows)
    b += batch * (2 * rows * h * hd * (2 if case["io"] == "bf16" else 4) + keys * kv8)
    return {"bytes": b, "flops": batch * 4 * h * hd * int((hi - lo).sum())}


# ------------------------------------------------------------------ inputs


def _inputs(case, seed):
    """Per batch slot: active positions, Q rows, the sequence's K and V rows and
    the active positions' fresh K and V rows (store and step), all f32 on the GPU.
    K has channels of unequal size, as after a trained projection, and V
    positions of unequal size."""
    h, hkv, hd = MODELS[case["model"]]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    slots = []
    for _ in range(case["batch"]):
        gain = torch.exp(0.4 * randn(hkv, hd))

        def rows(n):
            return randn(n, hkv, hd) * gain, randn(n, hkv, hd) * torch.exp(0.5 * randn(n, hkv, 1))

        s = {"pos": _positions(case, rng)}
        s["k"], s["v"] = rows(case["keys"])
        if case["op"] != "store":
            s["q"] = randn(case["rows"], h, hd)
            if case["io"] == "bf16":
                s["q"] = s["q"].bfloat16()
        if case["op"] != "attend":
            s["new_k"], s["new_v"] = rows(case["rows"])
        slots.append(s)
    return slots


_FRAMEWORK = {}


def _framework(io):
    """The framework's module and a program's context for these rows."""
    if not _FRAMEWORK:
        path = str(pathlib.Path(__file__).resolve().parent.parent / "diffuse-rs_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import dr_attn

        _FRAMEWORK["dr"] = dr_attn
        _FRAMEWORK["stream"] = torch.cuda.Stream()
    dr = _FRAMEWORK["dr"]
    if io not in _FRAMEWORK:
        ctx = dr.Context(torch.cuda.current_device())
        ctx.set_stream(_FRAMEWORK["stream"].cuda_stream)
        if io == "bf16":
            ctx.set_q_dtype(dr.DTYPE_BF16)
            ctx.set_o_dtype(dr.DTYPE_BF16)
        _FRAMEWORK[io] = ctx
    return dr, _FRAMEWORK[io]


def prepare(case, seed):
    """What a denoise loop has in hand before the call: the rows, and the cache
    with the sequence already in it (the plain form's cache is two tensors of
    codes and two of exponents)."""
    h, hkv, hd = MODELS[case["model"]]
    n, rows = case["keys"], case["rows"]
    state = {"case": case, "slots": _inputs(case, seed)}
    every = case["op"] == "store" and case["layout"] == "list"
    if own:
        dr, ctx = _framework(case["io"])
        cache = dr.StepCache(ctx, n, [hkv], [hd], n_batch=case["batch"], precision=[dr.PRECISION_FP8])
        whole = dr.Pass(ctx, range(n))
        torch.cuda.synchronize()
        for b, s in enumerate(state["slots"]):
            cache.store(0, whole, s["k"], s["v"], batch=b)
            s["pass"] = dr.Pass(ctx, s["pos"])
            if case["op"] != "attend":
                s["back"] = whole if every else s["pass"]
                s["out_k"], s["out_v"] = (torch.empty(n if every else rows, hkv, hd, device="cuda") for _ in range(2))
            if case["op"] != "store":
                s["out"] = torch.empty_like(s["q"])
        ctx.synchronize()
        state["cache"] = cache
        if case["op"] == "attend":
            state["items"] = [(s["q"], s["out"], s["pass"]) for s in state["slots"]]
        elif case["op"] == "step":
            state["items"] = [(s["q"], s["out"], s["pass"], s["new_k"], s["new_v"]) for s in state["slots"]]
    else:
        for s in state["slots"]:
            s["k8"], s["ke"] = _quantise(s["k"])
            s["v8"], s["ve"] = _quantise(s["v"])
            s["at"] = torch.from_numpy(s["pos"]).cuda()
            s["back"] = torch.arange(n, device="cuda") if every else s["at"]
    for s in state["slots"]:
        del s["k"], s["v"]
    return state


# ------------------------------------------------------------------ the operators


def run(state):
    case, slots = state["case"], state["slots"]
    h = MODELS[case["model"]][0]
    hd = MODELS[case["model"]][2]
    kw = {"sliding_window": case["window"] or None, "causal_prefix": case["prefix"] or None,
          "scale": 1.0 / math.sqrt(hd)}
    if own:
        cache = state["cache"]
        if case["op"] == "attend":
            cache.attention(0, state["items"], h, **kw)
            return [s["out"] for s in slots]
        if case["op"] == "step":
            cache.step(0, state["items"], h, **kw)
        else:
            for b, s in enumerate(slots):
                cache.store(0, s["pass"], s["new_k"], s["new_v"], batch=b)
        for b, s in enumerate(slots):
            cache.gather_pass(0, s["back"], s["out_k"], s["out_v"], batch=b)
        return [[s[x] for x in ("out", "out_k", "out_v") if x in s] for s in slots]
    return [_plain(case, s, **kw) for s in slots]


def _quantise(x):
    """Codes (e4m3) and exponents (int32) of f32 rows [n, heads, head_dim]."""
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))  # amax = m 2^e, m in [0.5, 1)
    e = torch.clamp(e - 9 + (m > 0.875).to(torch.int32), min=-126)
    return torch.ldexp(x, -e).to(torch.float8_e4m3fn), e


def _values(codes, e):
    return torch.ldexp(codes.float(), e)


def _plain(case, s, sliding_window, causal_prefix, scale):
    """One batch slot in elementary operations, 32 bits."""
    got = []
    if case["op"] != "attend":
        for x in ("k", "v"):
            codes, e = _quantise(s["new_" + x])
            s[x + "8"].view(torch.uint8).index_copy_(0, s["at"], codes.view(torch.uint8))
            s[x + "e"].index_copy_(0, s["at"], e)
            got.append(_values(s[x + "8"].view(torch.uint8).index_select(0, s["back"]).view(torch.float8_e4m3fn),
                               s[x + "e"].index_select(0, s["back"])))
    if case["op"] == "store":
        return got
    h, hkv, hd = MODELS[case["model"]]
    nq, group = case["rows"], h // hkv
    k = _values(s["k8"], s["ke"]).permute(1, 2, 0).contiguous()  # [hkv, hd, keys]
    v = _values(s["v8"], s["ve"]).permute(1, 0, 2).contiguous()  # [hkv, keys, hd]
    q = s["q"].float().reshape(nq, hkv, group, hd).permute(1, 2, 0, 3).reshape(hkv, group * nq, hd)
    sc = torch.matmul(q * scale, k).reshape(hkv, group, nq, case["keys"])
    if sliding_window or causal_prefix:
        qp, kp = s["at"][:, None], torch.arange(case["keys"], device="cuda")[None, :]
        hidden = torch.zeros(nq, case["keys"], dtype=torch.bool, device="cuda")
        if sliding_window:
            hidden |= (qp - kp).abs() >= sliding_window
        if causal_prefix:
            hidden |= (qp < causal_prefix) & (kp > qp)
        sc.masked_fill_(hidden, -math.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(hkv, group * nq, case["keys"]), v)
    o = o.reshape(hkv, group, nq, hd).permute(2, 0, 1, 3).reshape(nq, h, hd)
    return [o.to(s["q"].dtype).contiguous()] + got if case["op"] == "step" else o.to(s["q"].dtype).contiguous()


# ------------------------------------------------------------------ the definition, in 64 bits


def _e4m3_values(x):
    """The f64 values that rows x stand for once stored."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    # log2 may round to the next whole number just below a power of two
    e = torch.where(torch.exp2(e) > top, e - 1, e)
    e = torch.where(top / torch.exp2(e) > 1.75, e - 7, e - 8)
    unit = torch.exp2(torch.where(top > 0, torch.clamp(e, min=-126.0), torch.zeros_like(e)))
    y = x / unit
    mag = y.abs()
    g = torch.floor(torch.log2(torch.clamp(mag, min=2.0**-6)))
    g = torch.where(torch.exp2(g) > torch.clamp(mag, min=2.0**-6), g - 1, g)
    step = torch.exp2(g - 3)
    return torch.round(y / step) * step * unit  # (torch.round: half to even)


def exact(case, seed):
    h, hkv, hd = MODELS[case["model"]]
    n, nq = case["keys"], case["rows"]
    got = []
    for s in _inputs(case, seed):
        k, v = _e4m3_values(s["k"]), _e4m3_values(s["v"])
        at = torch.from_numpy(s["pos"]).cuda()
        back = []
        if case["op"] != "attend":
            k[at], v[at] = _e4m3_values(s["new_k"]), _e4m3_values(s["new_v"])
            back = [k, v] if case["op"] == "store" and case["layout"] == "list" else [k[at], v[at]]
        if case["op"] == "store":
            got.append(back)
            continue
        lo, hi = (torch.from_numpy(x).cuda()[:, None] for x in _band(case, s["pos"]))
        j = torch.arange(n, device="cuda")[None, :]
        sees = (j >= lo) & (j < hi)
        o = torch.empty(nq, h, hd, dtype=torch.float64, device="cuda")
        for head in range(h):
            g = head // (h // hkv)
            sc = (s["q"][:, head].double() @ k[:, g].t().contiguous()) / math.sqrt(hd)
            o[:, head] = torch.softmax(torch.where(sees, sc, -math.inf), -1) @ v[:, g].contiguous()
        got.append([o] + back if case["op"] == "step" else o)
    return got
