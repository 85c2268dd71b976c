"""The transformer-block operators together, as they are used: through the lazy device beside recorded work, as the layers of
the transformer, in captured and replayed serving steps, with two contexts and outgrown workspaces."""
import ctypes as C

import numpy as np
import pytest

import blockref as R
import devharness as H
import gpuharness as G
from aix_amd import device as D
from aix_amd import kernels as K
from oracle import cpuref as O
from oracle import drivers as OD

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = H.Dev()
    yield d
    d.close()


class OnDevice:
    """blockref.Box's idea of a GPU over the lazy device."""

    def __init__(self, dev):
        self.dev, self.ctx = dev, self

    def raw(self, nbytes):
        return self.dev.raw(nbytes)

    def upload(self, ptr, array):
        if array.nbytes:
            self.dev.dev.from_host(ptr, array)

    def download(self, array, ptr):
        self.dev.dev.to_host(array, ptr)


def box(gpu, dtype, shape, values=None, **kw):
    return R.Box(gpu, K, dtype, shape, values, **kw)


def ref(b):
    return C.byref(b.desc if isinstance(b, R.Box) else b)


def ptr(b):
    return C.pointer(b.desc)


@pytest.mark.parametrize("dtype", [O.F32, O.BF16])
def test_a_block_forward_and_backward_beside_recorded_work(dev, dtype):
    """x -> projection with bias -> rotary positions -> attention with a window -> projection with bias, SiLU and residual, and
    all the way back, through the device: operands that recorded operators produce, results that recorded operators read,
    fills that nobody has used yet, memory freed as soon as the program is done with it.  Every stage is checked against
    its definition on the values the device's previous stage left."""
    gpu = OnDevice(dev)
    call = dev.dev.call
    rng = np.random.default_rng(11)
    b, s, h, hk, d, window, sinks = 2, 37, 4, 2, 16, 12, 2
    t, e = b * s, h * d
    x0 = box(gpu, dtype, (t, e), rng.standard_normal((t, e)))
    half = np.array([0.5], np.float32)
    x, two = box(gpu, dtype, (t, e)), box(gpu, dtype, (t, e))
    call("fill", half.ctypes.data, O.F32, ref(two))
    call("mul", ref(x0), ref(two), ref(x))                                    # recorded: the first product has to wait for it
    weights = {n: (box(gpu, dtype, (i, o), rng.standard_normal((i, o)) * i ** -0.5), box(gpu, dtype, (1, o), rng.standard_normal((1, o)) * 0.1))
               for n, i, o in (("q", e, e), ("k", e, hk * d), ("v", e, hk * d), ("o", e, e))}
    zero = np.zeros(1, np.float32)

    def linear(inp, name, act, residual=None, keep=None):
        w, bias = weights[name]
        out = box(gpu, dtype, (inp.shape[0], w.shape[1]))
        call("fill", zero.ctypes.data, O.F32, ref(out))                       # a fill of the result that nobody reads: it must not land behind the product
        spec = K.Epilogue(bias=ptr(bias), residual=ptr(residual) if residual else None, pre=ptr(keep) if keep else None, activation=act)
        call("matmul_epilogue", ref(inp), ref(w), C.byref(spec), ref(out))
        return out

    def heads(flat, n):
        return K.tensor(flat.ptr, dtype, (b, n, s, d), (s * n * d, d, n * d, 1))

    def as_heads(flat, n):
        return flat.fetch().reshape(b, s, n, d).transpose(0, 2, 1, 3)

    q, k, v = (linear(x, n, K.ACT_NONE) for n in "qkv")
    pos_host = np.arange(s)[None] + np.array([[0], [50000]])
    pos = box(gpu, O.I32, (b, s), pos_host)
    tq, tk = box(gpu, dtype, (t, e)), box(gpu, dtype, (t, hk * d))
    turn = K.RotarySpec(dims=d, base=10000.0, factor=1.0, original_length=1.0, low_turns=1.0, high_turns=2.0, magnitude=1.0)
    call("rotary", C.byref(heads(q, h)), C.byref(heads(k, hk)), ref(pos), C.byref(turn), C.byref(heads(tq, h)), C.byref(heads(tk, hk)))
    lengths = box(gpu, O.I32, (b,), [s, 29])
    starts = box(gpu, O.I32, (b,), [0, 0])
    scale = float(np.float32(d ** -0.5))
    spec = K.AttentionSpec(scale=scale, causal=1, window=window, sinks=sinks, lengths=ptr(lengths), starts=ptr(starts))
    mixed, lse = box(gpu, dtype, (t, e)), box(gpu, O.F32, (b, h, s))
    call("attention", C.byref(heads(tq, h)), C.byref(heads(tk, hk)), C.byref(heads(v, hk)), C.byref(spec), C.byref(heads(mixed, h)), ref(lse))
    pre = box(gpu, dtype, (t, e))
    y = linear(mixed, "o", K.ACT_SILU, residual=x, keep=pre)
    grad = box(gpu, dtype, (t, e))
    call("sub", ref(y), ref(x), ref(grad))                                    # recorded: reads what the product just enqueued
    dz, dmixed, dw, dbias = box(gpu, dtype, (t, e)), box(gpu, dtype, (t, e)), box(gpu, dtype, (e, e)), box(gpu, dtype, (1, e))
    call("matmul_epilogue_backward", ref(grad), ref(mixed), ref(weights["o"][0]), ref(pre), K.ACT_SILU, ref(dz), ref(dmixed), ref(dw), ref(dbias))
    dq, dk, dv = box(gpu, dtype, (t, e)), box(gpu, dtype, (t, hk * d)), box(gpu, dtype, (t, hk * d))
    call("attention_backward", C.byref(heads(dmixed, h)), C.byref(heads(tq, h)), C.byref(heads(tk, hk)), C.byref(heads(v, hk)), C.byref(heads(mixed, h)), ref(lse),
         C.byref(spec), C.byref(heads(dq, h)), C.byref(heads(dk, hk)), C.byref(heads(dv, hk)))
    back = K.RotarySpec(dims=d, inverse=1, base=10000.0, factor=1.0, original_length=1.0, low_turns=1.0, high_turns=2.0, magnitude=1.0)
    dqx, dkx = box(gpu, dtype, (t, e)), box(gpu, dtype, (t, hk * d))
    call("rotary", C.byref(heads(dq, h)), C.byref(heads(dk, hk)), ref(pos), C.byref(back), C.byref(heads(dqx, h)), C.byref(heads(dkx, hk)))
    dev.free(two.ptr)                                                         # recorded work has used it, nothing else will
    dev.dev.synchronize()

    xv = x.fetch()
    for name, got in zip("qkv", (q, k, v)):
        w, bias = weights[name]
        want, far, _, _ = R.matmul_epilogue(xv, w.values(), bias.values(), None, "none", dtype)
        R.check(got.fetch(), want, far, "projection " + name)
    f = R.frequencies(d)
    for n, src, dst, inv in ((h, q, tq, 0), (hk, k, tk, 0), (h, dq, dqx, 1), (hk, dk, dkx, 1)):
        want, far = R.rotary(as_heads(src, n), pos_host, d, 0, inv, f, 1.0, dtype)
        R.check(as_heads(dst, n), want, far, "turn")
    seen = R.visible(b, s, s, True, window, sinks, [s, 29], [0, 0])
    out, want_lse, far, lse_far = R.attention(as_heads(tq, h), as_heads(tk, hk), as_heads(v, hk), seen, scale, dtype)
    R.check(as_heads(mixed, h), out, far, "attention")
    R.check(lse.fetch(), want_lse, lse_far, "lse")
    wo, bo = weights["o"]
    want, far, z, z_far = R.matmul_epilogue(mixed.fetch(), wo.values(), bo.values(), xv, "silu", dtype)
    R.check(y.fetch(), want, far, "output projection")
    R.check(pre.fetch(), z, z_far, "pre")
    assert np.array_equal(grad.fetch(), R.T_float(R.T_round((y.fetch() - xv).astype(np.float32), dtype), dtype))
    want, far = R.matmul_epilogue_backward(grad.fetch(), mixed.fetch(), wo.values(), pre.fetch(), "silu", dtype)
    for name, got, w_, f_ in zip(("dz", "dmixed", "dw", "dbias"), (dz, dmixed, dw, dbias), want, far):
        R.check(got.fetch().reshape(w_.shape), w_, f_, name)
    want, far = R.attention_backward(as_heads(dmixed, h), as_heads(tq, h), as_heads(tk, hk), as_heads(v, hk), as_heads(mixed, h), lse.fetch(), seen, scale, dtype)
    for name, got, n, w_, f_ in zip(("dq", "dk", "dv"), (dq, dk, dv), (h, hk, hk), want, far):
        R.check(as_heads(got, n), w_, f_, name)
    dev.live.remove(x.ptr)
    dev.dev.deallocate(x.ptr)
    dev.release()


def test_host_operands_are_staged_and_host_results_refused(dev):
    gpu = OnDevice(dev)
    rng = np.random.default_rng(4)
    a, b_ = rng.standard_normal((5, 24)).astype(np.float32), rng.standard_normal((24, 8)).astype(np.float32)
    bias = rng.standard_normal(8).astype(np.float32)
    ha, hb, hv = (K.tensor(m.ctypes.data, K.F32, m.shape) for m in (a, b_, bias))
    out = box(gpu, O.F32, (5, 8))
    spec = K.Epilogue(bias=C.pointer(hv), residual=None, pre=None, activation=K.ACT_RELU)
    dev.dev.call("matmul_epilogue", C.byref(ha), C.byref(hb), C.byref(spec), ref(out))
    want, far, _, _ = R.matmul_epilogue(a.astype(np.float64), b_.astype(np.float64), bias.astype(np.float64), None, "relu", O.F32)
    R.check(out.fetch(), want, far, "host operands")
    host = np.zeros((5, 8), np.float32)
    assert dev.dev.status("matmul_epilogue", C.byref(ha), C.byref(hb), C.byref(spec), C.byref(K.tensor(host.ctypes.data, K.F32, host.shape))) == 1
    assert b"must have GPU memory" in dev.dev.lib.aixhip_last_error()
    assert dev.dev.status("matmul_epilogue", C.byref(ha), C.byref(hb), None, ref(out)) == 1
    bad = K.RotarySpec(dims=3, base=1e4, magnitude=1.0)
    x = box(gpu, O.F32, (1, 1, 2, 8))
    p = box(gpu, O.I32, (1, 2))
    assert dev.dev.status("rotary", ref(x), None, ref(p), C.byref(bad), ref(x), None) == 1
    assert b"turned part" in dev.dev.lib.aixhip_last_error()
    dev.release()


@pytest.mark.parametrize("cfg", [(2, 64, 4, 32, 2, 128), (3, 128, 8, 64, 2, 256)], ids=str)
def test_the_transformer_on_blocks_against_the_cpu_device(dev, cfg):
    """Without window and rotary positions the layers compute what the composed program computes, with fewer roundings to bf16 on
    the way: the same bar as for the composed program on this device, 2e-2 against the CPU device with exact 16-bit sums."""
    from aix_amd import drivers as GD
    data = OD.transformer_data(*cfg)
    want_l, want_n, _ = OD.oracle_transformer(cfg, 1, data, threads=16, stacked=True, wide16=True)
    got_l, got_n, _, _ = GD.transformer_blocks(dev.dev, cfg, 2, data)
    big = want_n[0] > 1e-3 * want_n[0].max()
    rel = np.abs(got_n[0].astype(np.float64) - want_n[0])[big] / want_n[0][big]
    print(f"{cfg}: loss {want_l[0]:.6f} (cpu) {got_l[0]:.6f} (blocks); gradient norms max rel dev {rel.max():.2e}, median {np.median(rel):.2e}")
    assert np.all(np.isfinite(got_l)) and np.all(np.isfinite(got_n))
    assert abs(float(got_l[0]) - float(want_l[0])) <= 2e-2 * abs(float(want_l[0]))
    assert rel.max() <= 2e-2


def test_a_window_as_long_as_the_text_hides_nothing(dev):
    from aix_amd import drivers as GD
    cfg = (2, 128, 4, 96, 2, 128)
    data = OD.transformer_data(*cfg)
    plain_l, plain_n, _, _ = GD.transformer_blocks(dev.dev, cfg, 1, data)
    wide_l, wide_n, _, _ = GD.transformer_blocks(dev.dev, cfg, 1, data, window=96)
    kept_l, kept_n, _, _ = GD.transformer_blocks(dev.dev, cfg, 1, data, window=1, sinks=96)
    short_l, short_n, _, _ = GD.transformer_blocks(dev.dev, cfg, 1, data, window=8, sinks=1)
    assert plain_l[0] == wide_l[0] == kept_l[0] != short_l[0]
    assert np.array_equal(plain_n[:, 2:], wide_n[:, 2:]) and np.array_equal(plain_n[:, 2:], kept_n[:, 2:])
    assert np.all(np.isfinite(short_n))


def test_replays_of_a_captured_step_on_blocks_equal_the_eager_steps(dev):
    """As for the composed program: losses and gradient norms of the replays bit for bit (embedding gradients are summed with
    atomics: those two norms to 1e-3)."""
    from aix_amd import drivers as GD
    for cfg in ((2, 64, 4, 32, 2, 128), (1, 128, 4, 160, 3, 512)):
        data = OD.transformer_data(*cfg)
        eager_l, eager_n, _, _ = GD.transformer_blocks(dev.dev, cfg, 6, data, window=20, sinks=2, rotary_dims=cfg[1] // cfg[2])
        got_l, got_n, secs, nodes = GD.transformer_blocks(dev.dev, cfg, 6, data, window=20, sinks=2, rotary_dims=cfg[1] // cfg[2], capture_at=2)
        print(f"{cfg}: {nodes} graph nodes, replayed step {np.median(secs[3:]) * 1e3:.2f} ms")
        assert nodes > 10
        assert np.array_equal(got_l, eager_l)
        assert np.array_equal(got_n[:, 2:], eager_n[:, 2:])
        assert np.allclose(got_n[:, :2], eager_n[:, :2], rtol=1e-3, atol=0)


class Serving:
    """A single-token step on a context: rotary positions in place, attention over a cache, an output product."""

    def __init__(self, gpu, batch, keys, seed, window=300):
        rng = np.random.default_rng(seed)
        self.gpu, self.b, self.keys, self.h, self.hk, self.d, self.window = gpu, batch, keys, 8, 2, 64, window
        b, h, hk, d, e = batch, self.h, self.hk, self.d, self.h * self.d
        mk = lambda *shape: box(gpu, O.BF16, shape, rng.standard_normal(shape))      # noqa: E731
        self.q0 = mk(b, h, 1, d)
        self.k, self.v = (box(gpu, O.BF16, (b, hk, keys, d), rng.standard_normal((b, hk, keys, d)), order=(0, 2, 1, 3)) for _ in range(2))
        self.q, self.mixed = box(gpu, O.BF16, (b, h, 1, d)), box(gpu, O.BF16, (b, h, 1, d))
        self.pos, self.lengths = box(gpu, O.I32, (b, 1)), box(gpu, O.I32, (b,))
        self.w, self.bias, self.out = mk(e, 96), mk(96), box(gpu, O.BF16, (b, 96))
        self.turn = K.RotarySpec(dims=d, base=1e4, factor=1.0, original_length=1.0, low_turns=1.0, high_turns=2.0, magnitude=1.0)
        self.spec = K.AttentionSpec(scale=0.125, causal=1, window=window, sinks=4, lengths=ptr(self.lengths), starts=None)
        self.epi = K.Epilogue(bias=ptr(self.bias), residual=None, pre=None, activation=K.ACT_GELU)
        self.flat = K.tensor(self.mixed.ptr, K.BF16, (b, e))

    def at(self, lengths):
        self.lens = np.asarray(lengths)
        self.gpu.ctx.upload(self.lengths.ptr, self.lens.astype(np.int32))
        self.gpu.ctx.upload(self.pos.ptr, (self.lens - 1).astype(np.int32).reshape(-1, 1))

    def step(self):
        run = lambda name, *args: G.run_gpu(self.gpu, name, *args)               # noqa: E731
        run("aixk_rotary", ref(self.q0), None, ref(self.pos), C.byref(self.turn), ref(self.q), None)
        run("aixk_attention", ref(self.q), ref(self.k), ref(self.v), C.byref(self.spec), ref(self.mixed), None)
        run("aixk_matmul_epilogue", C.byref(self.flat), ref(self.w), C.byref(self.epi), ref(self.out))

    def check(self, what):
        pos = (self.lens - 1).reshape(-1, 1)
        want, far = R.rotary(self.q0.values(), pos, self.d, 0, 0, R.frequencies(self.d), 1.0, O.BF16)
        R.check(self.q.fetch(), want, far, what + " turn")
        seen = R.visible(self.b, 1, self.keys, True, self.window, 4, self.lens, None)
        out, _, far, _ = R.attention(self.q.fetch(), self.k.values(), self.v.values(), seen, 0.125, O.BF16)
        R.check(self.mixed.fetch(), out, far, what + " attention")
        want, far, _, _ = R.matmul_epilogue(self.mixed.fetch().reshape(self.b, -1), self.w.values(), self.bias.values(), None, "gelu", O.BF16)
        R.check(self.out.fetch(), want, far, what + " product")


def test_two_captured_serving_steps_share_their_context(dev):
    """Two steps of different sizes captured on one context, the workspaces outgrown by eager work in between, then replayed in
    turns with lengths and positions that move on: every replay follows the values in device memory."""
    gpu = G.Gpu()
    try:
        steps = [Serving(gpu, 2, 2000, 1), Serving(gpu, 3, 5000, 2)]
        graphs = []
        for n, s in enumerate(steps):
            s.at([s.keys] * s.b)
            s.step()
            s.check(f"eager {n}")
            gpu.ctx.call("aixk_capture_begin")
            s.step()
            g = C.c_void_p()
            gpu.ctx.call("aixk_capture_end", C.byref(g))
            graphs.append(g)
        big = Serving(gpu, 40, 3000, 3, window=2000)          # partial results of more rows than either captured step had
        big.at(np.linspace(1, 3000, 40).astype(int))
        big.step()
        big.check("eager, larger")
        rng = np.random.default_rng(9)
        a, b_ = (box(gpu, O.BF16, s, rng.standard_normal(s)) for s in ((130, 8192), (8192, 136)))
        prod = box(gpu, O.BF16, (130, 136))
        G.run_gpu(gpu, "aixk_matmul", ref(a), ref(b_), ref(prod))
        for turn in range(4):
            for n, s in enumerate(steps):
                s.at([1 + 317 * turn + 400 * i for i in range(s.b)])
                gpu.ctx.call("aixk_graph_launch", graphs[n])
                s.check(f"replay {turn} of {n}")
            big.step()
            big.check("eager, larger")
        for g in graphs:
            gpu.ctx.call("aixk_graph_destroy", g)
    finally:
        gpu.close()
        gpu.ctx.close()


def test_outgrown_workspaces_inside_a_capture_are_refused(dev):
    gpu = G.Gpu()
    try:
        s = Serving(gpu, 40, 3000, 3, window=2000)            # (a window of 300 is one workgroup's work and needs no workspace)
        s.at([3000] * 40)
        gpu.ctx.call("aixk_capture_begin")
        rc = gpu.ctx.lib.aixk_attention(gpu.ctx.handle, ref(s.q0), ref(s.k), ref(s.v), C.byref(s.spec), ref(s.mixed), None)
        text = gpu.ctx.lib.aixk_last_error().decode()
        gpu.ctx.call("aixk_capture_abort")
        assert rc == 1 and "inside a capture" in text
        s.step()
        s.check("afterwards")
    finally:
        gpu.close()
        gpu.ctx.close()


def test_two_contexts_at_once(dev):
    """Calls on two contexts of one GPU interleave; each has its own stream and workspaces."""
    gpus = [G.Gpu(), G.Gpu()]
    try:
        steps = [Serving(g, 4, 4000, 5 + n) for n, g in enumerate(gpus)]
        for n, s in enumerate(steps):
            s.at([4000, 17, 900, 2500 + n])
        for _ in range(20):
            for s in steps:
                s.step()
        for n, s in enumerate(steps):
            s.check(f"context {n}")
    finally:
        for g in gpus:
            g.close()
            g.ctx.close()
