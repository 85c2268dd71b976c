"""aixk_rotary against a plain 64-bit implementation: both pair layouts, a part of the head, scaled frequencies, far and
negative positions, one token and many, odd sizes and layouts, in place, and back again."""
import ctypes as C

import numpy as np
import pytest

import blockref as R
import gpuharness as G
from aix_amd import kernels as K
from oracle import cpuref as O

pytestmark = pytest.mark.gpu
SCALINGS = ["plain", "linear", "base", "parts"]


@pytest.fixture(scope="module")
def gpu():
    g = G.Gpu()
    yield g
    g.close()


def spec_of(dims, interleaved, inverse, scaling, magnitude, **kw):
    p = dict(base=10000.0, factor=4.0, original=2048.0, low=1.0, high=32.0)
    p.update(kw)
    spec = K.RotarySpec(dims=dims, interleaved=interleaved, inverse=inverse, scaling=SCALINGS.index(scaling), base=p["base"], factor=p["factor"],
                        original_length=p["original"], low_turns=p["low"], high_turns=p["high"], magnitude=magnitude)
    return spec, R.frequencies(dims, scaling, p["base"], p["factor"], p["original"], p["low"], p["high"])


def run(gpu, dtype, b, hq, hk, s, d, dims, interleaved=0, inverse=0, scaling="plain", magnitude=1.0, first=0, order=(0, 2, 1, 3), pad=0, offset=0, in_place=False,
        positions=None, **kw):
    rng = np.random.default_rng(b * 100 + s + d)
    spec, f = spec_of(dims, interleaved, inverse, scaling, magnitude, **kw)
    boxes = [R.Box(gpu, K, dtype, (b, h, s, d), rng.standard_normal((b, h, s, d)), order, pad, offset) for h in (hq, hk) if h is not None]
    outs = boxes if in_place else [R.Box(gpu, K, dtype, x.shape, None, order, pad, offset, 7.0) for x in boxes]
    at = first + np.arange(s)[None, :] + 1000 * np.arange(b)[:, None] if positions is None else np.asarray(positions)
    pos = R.Box(gpu, K, O.I32, (b, s), at)
    refs = [G.ref(x.desc) for x in boxes] + [None] * (2 - len(boxes))
    orefs = [G.ref(x.desc) for x in outs] + [None] * (2 - len(boxes))
    G.run_gpu(gpu, "aixk_rotary", refs[0], refs[1], G.ref(pos.desc), C.byref(spec), orefs[0], orefs[1])
    for x, y, name in zip(boxes, outs, "qk"):
        want, far = R.rotary(x.values(), at, dims, interleaved, inverse, f, magnitude, dtype)
        R.check(y.fetch(), want, far, name)
    gpu.release()


@pytest.mark.parametrize("dtype", [O.BF16, O.F16, O.F32])
@pytest.mark.parametrize("interleaved", [0, 1])
@pytest.mark.parametrize("d,dims", [(64, 64), (128, 64), (128, 128), (80, 20), (40, 40), (33, 6), (2, 2), (256, 256), (96, 90), (7, 4)])
def test_heads_and_parts(gpu, dtype, interleaved, d, dims):
    run(gpu, dtype, 2, 4, 2, 9, d, dims, interleaved)
    run(gpu, dtype, 3, 3, None, 1, d, dims, interleaved, inverse=1)


@pytest.mark.parametrize("dtype", [O.BF16, O.F32])
@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("first", [0, 120000, 2 ** 31 - 40000, -2 ** 31, -7])
def test_scaled_and_far(gpu, dtype, scaling, first):
    run(gpu, dtype, 2, 4, 1, 33, 128, 128, 0, 0, scaling, 1.2, first)
    run(gpu, dtype, 2, 4, 1, 33, 64, 32, 1, 1, scaling, 1.0, first, factor=0.5, base=500000.0)


@pytest.mark.parametrize("b,s,hq,hk", [(1, 1, 1, 1), (1, 1, 32, 8), (5, 1, 12, 12), (1, 4000, 3, 1), (3, 700, 16, 2), (2, 2, 200, 1), (1, 1, 0, 3), (2, 0, 4, 4), (0, 3, 4, 4)])
def test_sizes(gpu, b, s, hq, hk):
    run(gpu, O.F16, b, hq, hk, s, 64, 64)
    run(gpu, O.F16, b, hq, hk, s, 24, 10)


@pytest.mark.parametrize("dtype", [O.BF16, O.F32])
@pytest.mark.parametrize("order,pad,offset", [((0, 1, 2, 3), 0, 0), ((0, 2, 1, 3), 8, 16), ((0, 2, 1, 3), 3, 1), ((3, 0, 1, 2), 0, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_layouts_and_in_place(gpu, dtype, order, pad, offset, in_place):
    for interleaved in (0, 1):
        run(gpu, dtype, 2, 3, 2, 21, 64, 48, interleaved, order=order, pad=pad, offset=offset, in_place=in_place)


def test_shared_and_repeated_positions(gpu):
    run(gpu, O.BF16, 3, 2, 2, 4, 64, 64, positions=[[0, 0, 7, 7], [5, 5, 5, 5], [2 ** 31 - 1, -2 ** 31, 0, 1]])
    box = R.Box(gpu, K, O.F32, (3, 2, 4, 8), np.random.default_rng(0).standard_normal((3, 2, 4, 8)))
    out = R.Box(gpu, K, O.F32, (3, 2, 4, 8))
    row = R.Box(gpu, K, O.I32, (4,), [3, 1, 4, 1])
    shared = K.tensor(row.ptr, K.I32, (3, 4), (0, 1))                  # one row of positions for every sequence
    spec, f = spec_of(8, 0, 0, "plain", 1.0)
    G.run_gpu(gpu, "aixk_rotary", G.ref(box.desc), None, G.ref(shared), C.byref(spec), G.ref(out.desc), None)
    want, far = R.rotary(box.values(), np.tile([3, 1, 4, 1], (3, 1)), 8, 0, 0, f, 1.0, O.F32)
    R.check(out.fetch(), want, far, "one row of positions")
    gpu.release()


def test_the_inverse_is_the_gradient(gpu):
    """<turn(x), g> = <x, turn back(g)>: both sides in f32, off by the bounds of the two results."""
    rng = np.random.default_rng(2)
    x, g = (R.Box(gpu, K, O.F32, (2, 3, 50, 64), rng.standard_normal((2, 3, 50, 64))) for _ in range(2))
    y, h = (R.Box(gpu, K, O.F32, (2, 3, 50, 64)) for _ in range(2))
    pos = R.Box(gpu, K, O.I32, (2, 50), np.arange(100).reshape(2, 50) * 997)
    for inverse, src, dst in ((0, x, y), (1, g, h)):
        spec, f = spec_of(48, 1, inverse, "parts", 1.3)
        G.run_gpu(gpu, "aixk_rotary", G.ref(src.desc), None, G.ref(pos.desc), C.byref(spec), G.ref(dst.desc), None)
    _, far_y = R.rotary(x.values(), pos.values(), 48, 1, 0, f, 1.3, O.F32)
    _, far_h = R.rotary(g.values(), pos.values(), 48, 1, 1, f, 1.3, O.F32)
    left, right = (y.fetch() * g.values()).sum(), (x.values() * h.fetch()).sum()
    assert abs(left - right) <= (far_y * np.abs(g.values())).sum() + (far_h * np.abs(x.values())).sum()
    gpu.release()
