"""aixk_matmul_epilogue and its backward pass against plain 64-bit implementations: every route of the matrix product (few
rows, split sums, whole tiles, odd layouts), every part of the epilogue, in place."""
import ctypes as C

import numpy as np
import pytest

import blockref as R
import gpuharness as G
from aix_amd import kernels as K
from oracle import cpuref as O

pytestmark = pytest.mark.gpu
ACTS = ["none", "relu", "gelu", "silu"]
DTYPES = [O.BF16, O.F16, O.F32]


@pytest.fixture(scope="module")
def gpu():
    g = G.Gpu()
    yield g
    g.close()


def pointer(box):
    return C.pointer(box.desc) if box is not None else None


def ref(box):
    return G.ref(box.desc) if box is not None else None


def forward(gpu, dtype, m, k, n, act="gelu", bias=True, residual=True, keep=True, b_order=(0, 1), a_order=(0, 1), pad=0, offset=0, in_place=False, res_view=None):
    rng = np.random.default_rng(m + 7 * k + 13 * n)
    a = R.Box(gpu, K, dtype, (m, k), rng.standard_normal((m, k)), a_order, pad, offset)
    b = R.Box(gpu, K, dtype, (k, n), rng.standard_normal((k, n)) * max(k, 1) ** -0.5, b_order, pad, offset)
    v = R.Box(gpu, K, dtype, (n,), rng.standard_normal(n)) if bias else None
    r = R.Box(gpu, K, dtype, (m, n), rng.standard_normal((m, n)), pad=0 if in_place else pad, offset=0 if in_place else offset) if residual else None
    out = r if in_place else R.Box(gpu, K, dtype, (m, n), fill=7.0)
    pre = R.Box(gpu, K, dtype, (m, n), fill=7.0) if keep else None
    res_desc, res_values = (r.desc, r.values()) if r is not None else (None, None)
    if res_view == "row":                                   # one row for all
        res_desc, res_values = K.tensor(r.ptr, dtype, (m, n), (0, 1)), np.tile(r.values()[:1], (m, 1))
    spec = K.Epilogue(bias=pointer(v), residual=C.pointer(res_desc) if r is not None else None, pre=pointer(pre), activation=ACTS.index(act))
    G.run_gpu(gpu, "aixk_matmul_epilogue", ref(a), ref(b), C.byref(spec), ref(out))
    want, far, z, z_far = R.matmul_epilogue(a.values(), b.values(), v.values() if bias else None, res_values, act, dtype)
    R.check(out.fetch(), want, far, f"[{m}, {k}] x [{k}, {n}] {act}")
    if keep:
        R.check(pre.fetch(), z, z_far, f"[{m}, {k}] x [{k}, {n}] {act}: pre")
    gpu.release()


def backward(gpu, dtype, m, k, n, act="gelu", want_da=True, want_db=True, want_bias=True, pad=0, b_order=(0, 1), grad_order=(0, 1)):
    rng = np.random.default_rng(m + 7 * k + 13 * n)
    a = R.Box(gpu, K, dtype, (m, k), rng.standard_normal((m, k)), pad=pad)
    b = R.Box(gpu, K, dtype, (k, n), rng.standard_normal((k, n)) * max(n, 1) ** -0.5, b_order)
    grad = R.Box(gpu, K, dtype, (m, n), rng.standard_normal((m, n)), grad_order, pad)
    pre = R.Box(gpu, K, dtype, (m, n), rng.standard_normal((m, n)) * 2, grad_order, pad) if act != "none" else None
    dz = R.Box(gpu, K, dtype, (m, n), fill=7.0) if act != "none" else None
    da, db, dbias = R.Box(gpu, K, dtype, (m, k), fill=7.0), R.Box(gpu, K, dtype, (k, n), fill=7.0), R.Box(gpu, K, dtype, (n,), fill=7.0)
    G.run_gpu(gpu, "aixk_matmul_epilogue_backward", ref(grad), ref(a), ref(b), ref(pre), ACTS.index(act), ref(dz), ref(da) if want_da else None,
              ref(db) if want_db else None, ref(dbias) if want_bias else None)
    want, far = R.matmul_epilogue_backward(grad.values(), a.values(), b.values(), pre.values() if pre is not None else None, act, dtype)
    for box, w, f, name, on in zip((dz, da, db, dbias), want, far, ("dz", "da", "db", "dbias"), (dz is not None, want_da, want_db, want_bias)):
        if on:
            R.check(box.fetch(), w, f, f"[{m}, {k}] x [{k}, {n}] {act}: {name}")
        elif box is not None:
            assert np.all(box.fetch() == 7.0)
    gpu.release()


SHAPES = [(1, 1, 1), (1, 64, 8), (7, 768, 256), (16, 4096, 64), (3, 13, 5), (64, 64, 64), (130, 104, 72), (33, 13, 257), (100, 1000, 40), (128, 4096, 128), (300, 24, 300),
          (640, 128, 640), (1024, 64, 1024)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_sizes(gpu, dtype, m, k, n):
    forward(gpu, dtype, m, k, n)
    forward(gpu, dtype, m, k, n, "silu", residual=False, keep=False, b_order=(1, 0))


@pytest.mark.parametrize("dtype", [O.BF16, O.F16])
@pytest.mark.parametrize("m,k,n", [(2048, 64, 1024), (2048, 128, 1152), (4096, 64, 2048), (1280, 192, 1536)])
@pytest.mark.parametrize("b_order", [(0, 1), (1, 0)])
def test_whole_tiles(gpu, dtype, m, k, n, b_order):
    forward(gpu, dtype, m, k, n, b_order=b_order)


@pytest.mark.parametrize("dtype", [O.BF16, O.F16])
@pytest.mark.parametrize("m", [1, 7, 16, 17, 32, 33, 48, 64, 65])
@pytest.mark.parametrize("k,n", [(8, 8), (40, 56), (256, 33), (776, 2048), (4104, 64), (8192, 16), (520, 8200)])
@pytest.mark.parametrize("b_order", [(0, 1), (1, 0)])
def test_few_rows(gpu, dtype, m, k, n, b_order):
    forward(gpu, dtype, m, k, n, "silu", b_order=b_order)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,k,n", [(40, 72, 48), (9, 5, 11), (5, 8192, 64)])
def test_every_part(gpu, dtype, act, m, k, n):
    for bias in (False, True):
        for residual in (False, True):
            for keep in (False, True):
                forward(gpu, dtype, m, k, n, act, bias, residual, keep)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(70, 64, 96), (256, 256, 256), (5, 4096, 40), (1, 16, 8)])
def test_in_place_and_views(gpu, dtype, m, k, n):
    forward(gpu, dtype, m, k, n, in_place=True)
    forward(gpu, dtype, m, k, n, res_view="row")
    forward(gpu, dtype, m, k, n, pad=8, offset=16)
    forward(gpu, dtype, m, k, n, pad=3, offset=1)
    forward(gpu, dtype, m, k, n, a_order=(1, 0), pad=5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_to_sum_and_nothing_at_all(gpu, dtype):
    forward(gpu, dtype, 5, 0, 16)
    forward(gpu, dtype, 5, 0, 3, "silu")
    forward(gpu, dtype, 0, 8, 16)
    forward(gpu, dtype, 4, 8, 0)
    backward(gpu, dtype, 0, 8, 16)
    backward(gpu, dtype, 4, 8, 0)
    backward(gpu, dtype, 4, 0, 8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_far_arguments_of_the_activations(gpu, dtype):
    """Activations of zeros, tens and thousands (within the type): no overflow on the way, and the right limits."""
    near = np.array([0.0, -0.0, 1e-6, -1e-6, 3, -3, 9, -9, 12, -12, 40, -40, 300, -300, 6e4, -6e4])
    far = np.array([87, -87, 88.5, -88.5, 104, -104, 1e5, -1e5, 1e9, -1e9, 1e13, -1e13, 1e20, -1e20, 1e38, -1e38])
    for act, z in [(act, z) for act in ACTS for z in ((near,) if dtype == O.F16 else (near, far))]:
        a = R.Box(gpu, K, dtype, (1, 8))                     # a product of zeros: z is the bias
        b = R.Box(gpu, K, dtype, (8, 16))
        v = R.Box(gpu, K, dtype, (16,), z)
        out = R.Box(gpu, K, dtype, (1, 16))
        spec = K.Epilogue(bias=pointer(v), residual=None, pre=None, activation=ACTS.index(act))
        G.run_gpu(gpu, "aixk_matmul_epilogue", ref(a), ref(b), C.byref(spec), ref(out))
        want, _, far = R.activate(v.values(), act)
        R.check(out.fetch()[0], want, far + 4 * R.U32 * np.abs(want) + R.HALF[dtype] * np.abs(want) + R.TINY[dtype], act)
        if act != "none":
            pre, grad, dz = R.Box(gpu, K, dtype, (1, 16), z[None]), R.Box(gpu, K, dtype, (1, 16), np.ones((1, 16))), R.Box(gpu, K, dtype, (1, 16))
            G.run_gpu(gpu, "aixk_matmul_epilogue_backward", ref(grad), ref(a), ref(b), ref(pre), ACTS.index(act), ref(dz), None, None, None)
            s, s_far = R.slope(pre.values(), act)
            R.check(dz.fetch(), s, s_far + R.HALF[dtype] * np.abs(s) + R.TINY[dtype], act + " slope")
        gpu.release()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", SHAPES[:-2])
def test_backward_sizes(gpu, dtype, m, k, n):
    backward(gpu, dtype, m, k, n)
    backward(gpu, dtype, m, k, n, "none", pad=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_backward_parts(gpu, dtype, act):
    for want in ((True, False, False), (False, True, False), (False, False, True), (True, True, True)):
        backward(gpu, dtype, 65, 40, 48, act, *want)
    backward(gpu, dtype, 65, 40, 48, act, pad=3)
    backward(gpu, dtype, 65, 40, 48, act, b_order=(1, 0), grad_order=(1, 0))
    backward(gpu, dtype, 3000, 8, 24, act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 2, 7, 9, 31, 33, 65, 127, 1001, 4099])
@pytest.mark.parametrize("k,n", [(64, 64), (8, 16), (136, 264), (7, 24), (200, 65)])
def test_weight_gradients_of_any_number_of_rows(gpu, dtype, m, k, n):
    backward(gpu, dtype, m, k, n)


def test_gradients_against_differences(gpu):
    """f32: the directional derivative of sum(out w), by a central difference of the kernel's own forward pass with step 2^-7;
    the third derivative (step^2) and the rounding of the two sums stay below 2 % of the gradient's length."""
    rng = np.random.default_rng(3)
    m, k, n = 12, 20, 16
    boxes = {"a": R.Box(gpu, K, O.F32, (m, k), rng.standard_normal((m, k))), "b": R.Box(gpu, K, O.F32, (k, n), rng.standard_normal((k, n)) * 0.3),
             "bias": R.Box(gpu, K, O.F32, (n,), rng.standard_normal(n))}
    w, out, pre, dz = (R.Box(gpu, K, O.F32, (m, n), rng.standard_normal((m, n))) for _ in range(4))
    grads = {"a": R.Box(gpu, K, O.F32, (m, k)), "b": R.Box(gpu, K, O.F32, (k, n)), "bias": R.Box(gpu, K, O.F32, (n,))}
    for act in ("gelu", "silu"):
        spec = K.Epilogue(bias=pointer(boxes["bias"]), residual=None, pre=pointer(pre), activation=ACTS.index(act))
        run = lambda: G.run_gpu(gpu, "aixk_matmul_epilogue", ref(boxes["a"]), ref(boxes["b"]), C.byref(spec), ref(out))     # noqa: E731
        run()
        G.run_gpu(gpu, "aixk_matmul_epilogue_backward", ref(w), ref(boxes["a"]), ref(boxes["b"]), ref(pre), ACTS.index(act), ref(dz), ref(grads["a"]), ref(grads["b"]), ref(grads["bias"]))
        for name, box in boxes.items():
            way = rng.standard_normal(box.shape)
            way /= np.sqrt((way ** 2).sum())
            step, sums = 2.0 ** -7, []
            g = grads[name].fetch()
            for sign in (1, -1):
                store = box.before.copy()
                box.view(store)[...] = (box.values() + sign * step * way).astype(np.float32)
                gpu.ctx.upload(box.ptr, store)
                run()
                sums.append((out.fetch() * w.values()).sum())
            gpu.ctx.upload(box.ptr, box.before)
            assert abs((sums[0] - sums[1]) / (2 * step) - (g * way).sum()) <= 0.02 * np.sqrt((g ** 2).sum()), (act, name)
    gpu.release()
