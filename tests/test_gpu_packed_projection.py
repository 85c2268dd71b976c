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
