"""The operators on microscaled rows as a program calls them: a feed-forward in a
row, captured into a hipGraph and replayed, on two contexts at once, weights' slices,
the same bits again, offsets past 32 bits, the longest rows.  Needs an MI355X."""
from __future__ import annotations

import numpy as np
import pytest

import dr_attn as dr
import mx_reference as mx
from test_gpu_mx_matmul import acts, check_gated, product, weights
from test_gpu_mx_rows import FILL, empty_rows, get, get_rows, norm_error, norm_reference, put, put_rows
from test_gpu_parity import Dev, dev, say, torch  # noqa: F401

pytestmark = pytest.mark.gpu

EPS = 1e-5


class Block:
    """A layer's feed-forward: norm of x + residual, gated projections, down projection
    with the residual stream."""

    def __init__(self, dev, seed, n, cols, hidden, fmt=dr.MX_E4M3):
        rng = np.random.default_rng(seed)
        self.dev, self.n, self.cols, self.hidden, self.fmt = dev, n, cols, hidden, fmt
        self.x = mx.bf16(rng.standard_normal((n, cols)).astype(np.float32))
        self.res = mx.bf16((2 * rng.standard_normal((n, cols))).astype(np.float32))
        self.gain = rng.uniform(0.3, 3, cols).astype(np.float32)
        self.w = [weights(rng, hidden, cols), weights(rng, hidden, cols), weights(rng, cols, hidden)]
        self.dw = [put_rows(dev, *w, dr.MX_E2M1) for w in self.w]
        self.dx, self.dres, self.dgain = put(dev, self.x, True), put(dev, self.res, True), dev.put(self.gain)
        self.total, self.out = put(dev, np.zeros((n, cols), np.float32), True), put(dev, np.zeros((n, cols), np.float32), True)
        self.codes, self.mid = empty_rows(dev, n, cols, fmt), empty_rows(dev, n, hidden, fmt)

    def run(self, ctx=None):
        ctx, gate, up, down = ctx or self.dev.ctx, *self.dw
        dr.rms_norm_mx(ctx, self.dx, self.n, self.cols, self.codes, w=self.dgain, eps=EPS, residual=self.dres, total=self.total,
                       dtype=dr.DTYPE_BF16)
        dr.mx_gated(ctx, gate, up, self.hidden, self.cols, self.codes, self.n, self.mid)
        dr.mx_matmul(ctx, down, self.cols, self.hidden, self.mid, self.n, self.out, residual=self.total, dtype=dr.DTYPE_BF16)

    def results(self):
        """(sum, norm's codes, gated codes, out) as bytes."""
        return [self.dev.get(t).copy() for t in (self.total, self.codes.codes, self.codes.scales, self.mid.codes, self.mid.scales, self.out)]

    def check(self):
        """Each operator on what the one before it made."""
        n, cols, hidden = self.n, self.cols, self.hidden
        h, y = norm_reference(self.x, self.res, self.gain, EPS, True)
        assert np.array_equal(get(self.dev, self.total, True).reshape(n, cols), h)
        c, s = get_rows(self.dev, self.codes, n, cols)
        mx.check_codes(c, s, self.fmt, y, norm_error(y, cols))
        mc, ms = get_rows(self.dev, self.mid, n, hidden)
        check_gated(self.w[0], self.w[1], (c, s), self.fmt, cols, dr.ACT_SILU, mc, ms, self.fmt)
        want, _, tol = product(self.w[2], (mc, ms), self.fmt, hidden, False)
        err = np.abs(get(self.dev, self.out, True).reshape(n, cols) - (want + h))
        assert (err <= tol + 2.0**-8 * (np.abs(want + h) + tol)).all()


@pytest.mark.parametrize("fmt", [dr.MX_E4M3, dr.MX_E2M1], ids=["8bit", "4bit"])
@pytest.mark.parametrize("n,cols,hidden", [(1, 2048, 1024), (7, 672, 1120), (96, 2048, 1024), (300, 544, 1536)])
def test_feed_forward(dev, fmt, n, cols, hidden):
    say(f"feed-forward n {n} cols {cols} hidden {hidden} fmt {fmt}")
    b = Block(dev, n + cols, n, cols, hidden, fmt)
    b.run()
    b.check()
    first = b.results()
    b.run()
    assert all(np.array_equal(x, y) for x, y in zip(first, b.results()))  # the same bits again


def test_graph(dev):
    """A captured feed-forward, replayed with new inputs and with other work between."""
    t = dev.t
    b, other = Block(dev, 1, 33, 1024, 1536), Block(dev, 2, 1, 2048, 1024)
    b.run()
    other.run()
    dev.stream.synchronize()
    allocs = dr.alloc_count()
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g, stream=dev.stream):
        b.run()
        other.run()
    assert dr.alloc_count() == allocs
    for k in range(4):
        rng = np.random.default_rng(10 + k)
        b.x = mx.bf16(rng.standard_normal(b.x.shape).astype(np.float32) * (1 + k))
        with t.cuda.stream(dev.stream):
            b.dx.copy_(put(dev, b.x, True))
            for x in (b.codes.codes, b.mid.codes, other.mid.codes):
                x.fill_(FILL)
        dev.stream.synchronize()
        with t.cuda.stream(dev.stream):
            g.replay()
        b.check()
        other.check()
        got = b.results()
        b.run()  # eagerly, between two replays
        assert all(np.array_equal(x, y) for x, y in zip(got, b.results()))


def test_two_contexts(torch):
    """Two contexts on two streams, their calls interleaved and nothing waited for."""
    devs = [Dev(torch), Dev(torch)]
    blocks = [Block(d, 5 + i, 40 + 100 * i, 1024, 1536) for i, d in enumerate(devs)]
    torch.cuda.synchronize()
    for _ in range(5):
        for b in blocks:
            b.run()
    for b in blocks:
        b.check()


def test_stream_switch(dev, torch):
    """A context's next stream waits for what the last one holds."""
    b = Block(dev, 9, 64, 2048, 1536)
    ctx, second = dr.Context(0), torch.cuda.Stream()
    ctx.set_stream(dev.stream.cuda_stream)
    dev.stream.synchronize()
    gate, up, down = b.dw
    dr.rms_norm_mx(ctx, b.dx, b.n, b.cols, b.codes, w=b.dgain, eps=EPS, residual=b.dres, total=b.total, dtype=dr.DTYPE_BF16)
    dr.mx_gated(ctx, gate, up, b.hidden, b.cols, b.codes, b.n, b.mid)
    ctx.set_stream(second.cuda_stream)
    dr.mx_matmul(ctx, down, b.cols, b.hidden, b.mid, b.n, b.out, residual=b.total, dtype=dr.DTYPE_BF16)
    second.synchronize()
    b.check()


def test_slice_of_weights(dev):
    """An expert's rows of a stack, by the planes' addresses."""
    rng = np.random.default_rng(3)
    rows, cols, n, experts = 96, 544, 20, 5
    w, a = weights(rng, rows * experts, cols), acts(rng, n, cols, dr.MX_E4M3)
    stack, da = put_rows(dev, *w, dr.MX_E2M1), put_rows(dev, *a, dr.MX_E4M3)
    for e in (0, 3, 4):
        part = dr.MxRows(stack.codes.data_ptr() + e * rows * cols // 2, stack.scales.data_ptr() + e * rows * dr.mx_pitch(cols), dr.MX_E2M1)
        out = dev.empty(n * rows)
        dr.mx_matmul(dev.ctx, part, rows, cols, da, n, out)
        s, _, tol = product((w[0][e * rows:(e + 1) * rows], w[1][e * rows:(e + 1) * rows]), a, dr.MX_E4M3, cols, True)
        assert (np.abs(dev.get(out).reshape(n, rows) - s) <= tol + 2.0**-24 * np.abs(s)).all()


def test_any_alignment_of_out(dev):
    """out and residual at odd elements: the same values as at aligned ones."""
    rng = np.random.default_rng(4)
    for n, rows, cols in ((5, 64, 96), (40, 96, 160), (513, 1032, 544)):
        w, a = weights(rng, rows, cols), acts(rng, n, cols, dr.MX_E4M3)
        dw, da = put_rows(dev, *w, dr.MX_E2M1), put_rows(dev, *a, dr.MX_E4M3)
        res = mx.bf16(rng.standard_normal(n * rows + 1).astype(np.float32))
        for bf16 in (False, True):
            size, dtype = (2, dr.DTYPE_BF16) if bf16 else (4, dr.DTYPE_F32)
            dres, odd, even = put(dev, res, bf16), put(dev, np.full(n * rows + 2, 7.0), bf16), put(dev, np.zeros(n * rows), bf16)
            dr.mx_matmul(dev.ctx, dw, rows, cols, da, n, odd.data_ptr() + size, residual=dres.data_ptr() + size, dtype=dtype)
            aligned = put(dev, res[1:], bf16)
            dr.mx_matmul(dev.ctx, dw, rows, cols, da, n, even, residual=aligned, dtype=dtype)
            got = get(dev, odd, bf16)
            assert got[0] == 7 and got[-1] == 7
            assert np.array_equal(got[1:-1], get(dev, even, bf16))


@pytest.mark.parametrize("fmt", [dr.MX_E4M3, dr.MX_E2M1], ids=["8bit", "4bit"])
def test_longest_rows(dev, fmt):
    """2^22 columns: the kernels' 32-bit offsets within a tile."""
    t = dev.t
    cols, rows, n = 1 << 22, 20, 18
    rng = np.random.default_rng(6)
    step = rng.integers(0, 2, (rows, cols // 32)).astype(np.uint8)  # (values of every size, made quickly)
    wc = rng.integers(0, 256, (rows, cols // 2), dtype=np.uint8)
    ac = rng.integers(0, 120, (n, cols // 2 if fmt == dr.MX_E2M1 else cols), dtype=np.uint8)
    ws, as_ = (124 + step).astype(np.uint8), np.full((n, cols // 32), 120, np.uint8)
    want = []
    with t.cuda.stream(dev.stream):
        wv, av = (t.from_numpy(mx.values(c, s, f, cols).astype(np.float32)).cuda().double()
                  for c, s, f in ((wc, ws, dr.MX_E2M1), (ac, as_, fmt)))
        want, p = (av @ wv.t().contiguous()).cpu().numpy(), (av.abs() @ wv.abs().t().contiguous()).cpu().numpy()
        del wv, av
    dw, da = put_rows(dev, wc, ws, dr.MX_E2M1), put_rows(dev, ac, as_, fmt)
    for m in (1, n):
        out = dev.empty(m * rows)
        dr.mx_matmul(dev.ctx, dw, rows, cols, da, m, out)
        err = np.abs(dev.get(out).reshape(m, rows) - want[:m])
        assert (err <= 4 * np.sqrt(cols) * 2.0**-23 * p[:m] + 2.0**-24 * np.abs(want[:m])).all()


def test_norm_of_the_longest_row(dev):
    cols = 1 << 22
    rng = np.random.default_rng(8)
    x = rng.standard_normal((1, cols)).astype(np.float32)
    out = empty_rows(dev, 1, cols, dr.MX_E4M3)
    dr.rms_norm_mx(dev.ctx, dev.put(x), 1, cols, out, eps=EPS)
    _, y = norm_reference(x, None, None, EPS, False)
    mx.check_codes(*get_rows(dev, out, 1, cols), dr.MX_E4M3, y, norm_error(y, cols))


def test_offsets_past_32_bits(dev):
    """2.3e9 outputs, and as many values quantised: their last rows."""
    t = dev.t
    n, rows, cols = 70016, 32800, 32
    rng = np.random.default_rng(7)
    w, a = weights(rng, rows, cols), acts(rng, n, cols, dr.MX_E2M1)
    dw, da = put_rows(dev, *w, dr.MX_E2M1), put_rows(dev, *a, dr.MX_E2M1)
    with t.cuda.stream(dev.stream):
        out = t.zeros(n, rows, dtype=t.bfloat16, device="cuda")
    say(f"product of {n} x {rows}")
    dr.mx_matmul(dev.ctx, dw, rows, cols, da, n, out, dtype=dr.DTYPE_BF16)
    dev.stream.synchronize()
    for lo in (0, n // 2, n - 40):
        s, _, tol = product(w, (a[0][lo:lo + 40], a[1][lo:lo + 40]), dr.MX_E2M1, cols, True)
        got = out[lo:lo + 40].float().cpu().numpy()
        assert (np.abs(got - s) <= tol + 2.0**-8 * (np.abs(s) + tol)).all()
    say("quantised and read back")
    codes = t.empty(n * rows // 2, dtype=t.uint8, device="cuda")
    q = dr.MxRows(codes, t.empty(n * dr.mx_pitch(rows), dtype=t.uint8, device="cuda"), dr.MX_E2M1)
    dr.mx_quantize(dev.ctx, out, n, rows, q, dtype=dr.DTYPE_BF16)
    dev.stream.synchronize()
    last = out[-3:].float().cpu().numpy()
    c, s = mx.quantise(last, dr.MX_E2M1)
    assert np.array_equal(codes[-3 * (rows // 2):].cpu().numpy().reshape(3, -1), c)
    dr.mx_dequantize(dev.ctx, q, n, rows, out, dtype=dr.DTYPE_BF16)
    dev.stream.synchronize()
    assert np.array_equal(out[-3:].float().cpu().numpy(), mx.values(c, s, dr.MX_E2M1, rows))
    say("normed")
    total = t.empty_like(out)
    dr.rms_norm_mx(dev.ctx, out, n, rows, q, residual=out, total=total, dtype=dr.DTYPE_BF16)
    dev.stream.synchronize()
    h, y = norm_reference(out[-2:].float().cpu().numpy(), out[-2:].float().cpu().numpy(), None, 1e-6, True)
    assert np.array_equal(total[-2:].float().cpu().numpy(), h)
    got_s = q.scales[-2 * dr.mx_pitch(rows):].cpu().numpy().reshape(2, -1)
    mx.check_codes(codes[-2 * (rows // 2):].cpu().numpy().reshape(2, -1), got_s, dr.MX_E2M1, y, norm_error(y, rows))
