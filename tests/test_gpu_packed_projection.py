"""Queries, keys and values as one projection leaves them, side by side in its rows: turned in place, attended to, and their
gradients written side by side again.  Bounds: blockref.py."""
import ctypes as C

import numpy as np
import pytest

import blockref as R
import gpuharness as G
from aix_amd import kernels as K
from oracle import cpuref as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    g = G.Gpu()
    yield g
    g.close()


class Packed:
    """[batch, length, (sum of heads) d + gap] of one element type with views [batch, heads, length, d] in it."""

    def __init__(self, gpu, dtype, batch, length, heads, d, gap, values=None):
        self.gpu, self.dtype, self.heads, self.d = gpu, dtype, heads, d
        self.width = sum(heads) * d + gap
        self.shape = (batch, length, self.width)
        values = np.full(self.shape, 7.0) if values is None else values
        self.store = R.T_round(values, dtype).reshape(self.shape)
        self.ptr = gpu.raw(self.store.nbytes)
        gpu.ctx.upload(self.ptr, self.store)
        self.at = [sum(heads[:n]) * d for n in range(len(heads))]
        strides = (length * self.width, d, self.width, 1)
        self.views = [K.tensor(self.ptr, dtype, (batch, h, length, d), strides, at) for h, at in zip(heads, self.at)]

    def part(self, store, n):
        x = R.T_float(store[:, :, self.at[n]:self.at[n] + self.heads[n] * self.d], self.dtype)
        return x.reshape(*self.shape[:2], self.heads[n], self.d).transpose(0, 2, 1, 3)

    def fetch(self):
        raw = np.empty_like(self.store)
        self.gpu.ctx.download(raw, self.ptr)
        return raw


@pytest.mark.parametrize("dtype", [O.BF16, O.F16, O.F32])
@pytest.mark.parametrize("batch,length,heads,d", [(2, 70, (4, 2, 2), 64), (1, 1, (3, 3, 3), 32), (3, 5, (2, 1, 1), 40)])
def test_turned_in_place_attended_and_back(gpu, dtype, batch, length, heads, d):
    rng = np.random.default_rng(length + d)
    gap = 16
    p = Packed(gpu, dtype, batch, length, heads, d, gap, rng.standard_normal((batch, length, sum(heads) * d + gap)))
    positions = np.tile(np.arange(length, dtype=np.int32) + 5, (batch, 1))
    where = R.Box(gpu, K, O.I32, positions.shape, positions)
    spec = K.RotarySpec(dims=d - d % 8, interleaved=0, inverse=0, scaling=K.ROTARY_PLAIN, base=1e4, factor=1.0, original_length=1.0, low_turns=0.0, high_turns=1.0, magnitude=1.0)
    q, k, v = p.views
    G.run_gpu(gpu, "aixk_rotary", G.ref(q), G.ref(k), G.ref(where.desc), C.byref(spec), G.ref(q), G.ref(k))
    got = p.fetch()
    for n in (0, 1):
        want, far = R.rotary(p.part(p.store, n), positions, spec.dims, False, False, R.frequencies(spec.dims), 1.0, dtype)
        R.check(p.part(got, n), want, far, f"turned in place, part {n}")
    assert np.array_equal(got[:, :, p.at[2]:], p.store[:, :, p.at[2]:]), "values or what lies behind them were written"

    turned = [p.part(got, n) for n in range(3)]
    out, grad = R.Box(gpu, K, dtype, (batch, heads[0], length, d)), R.Box(gpu, K, dtype, (batch, heads[0], length, d), rng.standard_normal((batch, heads[0], length, d)))
    lse = R.Box(gpu, K, O.F32, (batch, heads[0], length))
    mask = K.AttentionSpec(scale=d ** -0.5, causal=1, window=0, sinks=0, lengths=None, starts=None)
    G.run_gpu(gpu, "aixk_attention", G.ref(q), G.ref(k), G.ref(v), C.byref(mask), G.ref(out.desc), G.ref(lse.desc))
    back = Packed(gpu, dtype, batch, length, heads, d, gap)
    G.run_gpu(gpu, "aixk_attention_backward", G.ref(grad.desc), G.ref(q), G.ref(k), G.ref(v), G.ref(out.desc), G.ref(lse.desc), C.byref(mask), *[G.ref(t) for t in back.views])
    gpu.ctx.sync()
    seen = R.visible(batch, length, length, True, 0, 0, None, None)
    scale = float(np.float32(mask.scale))
    want, _, far, _ = R.attention(*turned, seen, scale, dtype)
    R.check(out.fetch(), want, far, "out")
    want, far = R.attention_backward(grad.values(), *turned, out.fetch(), lse.fetch(), seen, scale, dtype)
    raw = back.fetch()
    for n, name in enumerate(("dq", "dk", "dv")):
        R.check(back.part(raw, n), want[n], far[n], name)
    assert np.all(R.T_float(raw[:, :, back.width - gap:], dtype) == 7.0), "what lies behind the gradients was written"
    gpu.release()


@pytest.mark.parametrize("dtype", [O.BF16, O.F16])
def test_a_training_step_on_packed_parts_captured_and_replayed(gpu, dtype):
    """Projection, turn in place, attention with leading keys that have shares of their own, and the gradients side by side: captured
    once, replayed on other inputs with eager calls in between, each replay equal to the eager step bit for bit."""
    rng = np.random.default_rng(4)
    batch, length, heads, d = 1, 1500, (2, 2, 2), 64
    rows, width, inner = batch * length, sum(heads) * d, 96
    shape = (batch, heads[0], length, d)
    box = lambda s, v=None: R.Box(gpu, K, dtype, s, v)                                # noqa: E731
    x, w, bias = box((rows, inner)), box((inner, width), rng.standard_normal((inner, width)) * inner ** -0.5), box((1, width), rng.standard_normal((1, width)))
    p, back = Packed(gpu, dtype, batch, length, heads, d, 0), Packed(gpu, dtype, batch, length, heads, d, 0)
    flat, flat_back = (K.tensor(t.ptr, dtype, (rows, width)) for t in (p, back))
    out, grad, lse = box(shape), box(shape), R.Box(gpu, K, O.F32, shape[:3])
    dx, dw, db = box((rows, inner)), box((inner, width)), box((1, width))
    positions = R.Box(gpu, K, O.I32, (batch, length), np.arange(length)[None])
    turn, turn_back = (K.RotarySpec(dims=d, inverse=n, base=1e4, factor=1.0, original_length=1.0, low_turns=0.0, high_turns=1.0, magnitude=1.0) for n in (0, 1))
    mask = K.AttentionSpec(scale=0.125, causal=1, window=50, sinks=400, lengths=None, starts=None)
    epilogue = K.Epilogue(bias=C.pointer(bias.desc), residual=None, pre=None, activation=K.ACT_NONE)
    run = lambda name, *args: G.run_gpu(gpu, name, *args)                             # noqa: E731

    def step():
        run("aixk_matmul_epilogue", G.ref(x.desc), G.ref(w.desc), C.byref(epilogue), G.ref(flat))
        run("aixk_rotary", G.ref(p.views[0]), G.ref(p.views[1]), G.ref(positions.desc), C.byref(turn), G.ref(p.views[0]), G.ref(p.views[1]))
        run("aixk_attention", *[G.ref(t) for t in p.views], C.byref(mask), G.ref(out.desc), G.ref(lse.desc))
        run("aixk_attention_backward", G.ref(grad.desc), *[G.ref(t) for t in p.views], G.ref(out.desc), G.ref(lse.desc), C.byref(mask), *[G.ref(t) for t in back.views])
        run("aixk_rotary", G.ref(back.views[0]), G.ref(back.views[1]), G.ref(positions.desc), C.byref(turn_back), G.ref(back.views[0]), G.ref(back.views[1]))
        run("aixk_matmul_epilogue_backward", G.ref(flat_back), G.ref(x.desc), G.ref(w.desc), None, K.ACT_NONE, None, G.ref(dx.desc), G.ref(dw.desc), G.ref(db.desc))

    def put(seed):
        r = np.random.default_rng(seed)
        gpu.ctx.upload(x.ptr, R.T_round(r.standard_normal(x.shape), dtype))
        gpu.ctx.upload(grad.ptr, R.T_round(r.standard_normal(shape) * 2.0 ** (seed % 5), dtype))

    def results():
        gpu.ctx.sync()
        return [b.fetch().tobytes() for b in (out, lse, dx, dw, db)] + [p.fetch().tobytes(), back.fetch().tobytes()]

    put(0)
    step()
    first = results()
    gpu.ctx.call("aixk_capture_begin")
    step()
    graph = C.c_void_p()
    gpu.ctx.call("aixk_capture_end", C.byref(graph))
    for seed in (1, 2, 3, 0):
        put(seed)
        step()
        eager = results()
        gpu.ctx.upload(out.ptr, np.zeros_like(out.store))
        gpu.ctx.upload(back.ptr, np.zeros_like(back.store))
        gpu.ctx.call("aixk_graph_launch", graph)
        assert results() == eager, f"replay on inputs {seed}"
    assert eager == first and np.isfinite(dw.fetch()).all()
    gpu.ctx.call("aixk_graph_destroy", graph)
    gpu.release()


def test_packed_parts_through_the_device():
    """The same turn and attention through the lazy device: the projection's sum is recorded, the turn in place waits for it."""
    import devharness as H
    from test_gpu_block_operators import OnDevice
    dev = H.Dev()
    gpu = OnDevice(dev)
    rng = np.random.default_rng(8)
    batch, length, heads, d = 2, 33, (4, 2, 2), 32
    dtype, width = O.BF16, sum(heads) * d
    shape = (batch, length, width)
    a, b, total = (R.Box(gpu, K, dtype, shape, v) for v in (rng.standard_normal(shape), rng.standard_normal(shape), None))
    dev.dev.call("add", G.ref(a.desc), G.ref(b.desc), G.ref(total.desc))
    strides = (length * width, d, width, 1)
    q, k, v = (K.tensor(total.ptr, dtype, (batch, h, length, d), strides, at) for h, at in zip(heads, (0, 4 * d, 6 * d)))
    positions = R.Box(gpu, K, O.I32, (batch, length), np.tile(np.arange(length), (batch, 1)))
    turn = K.RotarySpec(dims=d, base=1e4, factor=1.0, original_length=1.0, low_turns=0.0, high_turns=1.0, magnitude=1.0)
    dev.dev.call("rotary", G.ref(q), G.ref(k), G.ref(positions.desc), C.byref(turn), G.ref(q), G.ref(k))
    mask = K.AttentionSpec(scale=0.25, causal=1, window=0, sinks=0, lengths=None, starts=None)
    out = R.Box(gpu, K, dtype, (batch, heads[0], length, d))
    dev.dev.call("attention", G.ref(q), G.ref(k), G.ref(v), C.byref(mask), G.ref(out.desc), None)
    dev.dev.synchronize()
    start = R.T_float(R.T_round((a.values() + b.values()).astype(np.float32), dtype), dtype)
    got = total.fetch()
    part = lambda y, n, h: y[:, :, n * d:(n + h) * d].reshape(batch, length, h, d).transpose(0, 2, 1, 3)      # noqa: E731
    for n, h in ((0, 4), (4, 2)):
        want, far = R.rotary(part(start, n, h), np.tile(np.arange(length), (batch, 1)), d, False, False, R.frequencies(d), 1.0, dtype)
        R.check(part(got, n, h), want, far, "turn")
    assert np.array_equal(part(got, 6, 2), part(start, 6, 2))
    want, _, far, _ = R.attention(part(got, 0, 4), part(got, 4, 2), part(got, 6, 2), R.visible(batch, length, length, True, 0, 0, None, None), 0.25, dtype)
    R.check(out.fetch(), want, far, "attention")
    dev.release()
    dev.close()
