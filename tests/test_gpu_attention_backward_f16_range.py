"""The gradients of attention in f16 where dS = P (grad v^T - delta) or P leave f16's range though operands and gradients do not:
loss-scaled gradients, small ones, and even rows over many keys.

Bounds as in blockref.py, but where that allows f16's smallest step per pair: P is at most 1 and kept times 2^15, so it is off by
half a step at that scale, 2^-25 2^-15; dS of a query (for dq) or a key (for dk) is kept in a unit in which the largest one of its tile
came to 2^11 at least, so it is off by 2^-25 2^-11 of the largest dS of that query or key."""
import numpy as np
import pytest

import blockref as R
import gpuharness as G
from oracle import cpuref as O

from test_gpu_attention import Case

pytestmark = pytest.mark.gpu
H, TINY, U32, FLUSH = R.HALF[O.F16], R.TINY[O.F16], R.U32, R.FLUSH


@pytest.fixture(scope="module")
def gpu():
    g = G.Gpu()
    yield g
    g.close()


def gradients(case):
    q, k, v, grad, out, lse = (b.fetch() if b in (case.out, case.lse) else b.values() for b in (case.q, case.k, case.v, case.grad, case.out, case.lse))
    group, d = q.shape[1] // k.shape[1], q.shape[3]
    got, far = [np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)], [np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)]
    for b in range(q.shape[0]):
        for c in range(k.shape[1]):
            rows, most = [], np.zeros(k.shape[2])
            for h in range(c * group, (c + 1) * group):
                ok, kk, vv, qq, gg, yy = case.seen[b], k[b, c], v[b, c], q[b, h], grad[b, h], out[b, h]
                stat = np.where(np.isfinite(lse[b, h]), lse[b, h], np.inf)[:, None]
                w = np.where(ok, np.exp(np.minimum(case.scale * (qq @ kk.T) - stat, 700)), 0)
                dp, delta = gg @ vv.T, (gg * yy).sum(1)[:, None]
                ds = w * (dp - delta)
                e = R.score_far(qq, kk, case.scale, ok, d)[:, None] + 4 * U32 * np.abs(np.where(np.isfinite(stat), stat, 0))
                dp_far = (d + 4) * U32 * (np.abs(gg) @ np.abs(vv).T + (np.abs(gg) * np.abs(yy)).sum(1)[:, None])
                rows.append((h, ok, w, ds, (H + e) * w + (FLUSH + 2.0 ** -40) * ok, (H + e + 4 * U32) * np.abs(ds) + w * dp_far + FLUSH * (1 + np.abs(dp - delta)) * ok))
                most = np.maximum(most, np.abs(ds).max(0))
            for h, ok, w, ds, w_far, ds_far in rows:
                of_row = ds_far + 2.0 ** -36 * np.abs(ds).max(1)[:, None] * ok
                of_key = ds_far + 2.0 ** -36 * most * ok
                qq, gg = q[b, h], grad[b, h]
                nk, nq = ok.sum(1)[:, None], (ok.sum(0) * group)[:, None]
                got[0][b, h] = case.scale * (ds @ k[b, c])
                got[1][b, c] += case.scale * (ds.T @ qq)
                got[2][b, c] += w.T @ gg
                far[0][b, h] = case.scale * (of_row @ np.abs(k[b, c]) + (nk + 8) * U32 * (np.abs(ds) @ np.abs(k[b, c])))
                far[1][b, c] += case.scale * (of_key.T @ np.abs(qq) + (nq + 8) * U32 * (np.abs(ds).T @ np.abs(qq)))
                far[2][b, c] += w_far.T @ np.abs(gg) + (nq + 8) * U32 * (w.T @ np.abs(gg))
    return got, [f + H * np.abs(g) + TINY for f, g in zip(far, got)]


def change(case, box, values):
    store = box.before.copy()
    box.view(store)[...] = R.T_round(values, O.F16)
    box.before = store
    case.gpu.ctx.upload(box.ptr, store)


def check(case, what):
    case.forward()
    case.check_forward(what)
    case.backward()
    case.gpu.ctx.sync()
    want, far = gradients(case)
    for n, (box, name) in enumerate(zip((case.dq, case.dk, case.dv), ("dq", "dk", "dv"))):
        R.check(box.fetch(), want[n], far[n], f"{what} {name}")
    return want


@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_score_gradient_beyond_f16(gpu, d):
    """Two keys of even weight: dS = 64 d 32 / 2 = 65536 at 64 dims, more above; its products with the keys cancel to what f16 holds."""
    case = Case(gpu, O.F16, 1, 1, 1, 1, 2, d, causal=False)
    change(case, case.q, np.zeros((1, 1, 1, d)))
    change(case, case.grad, np.full((1, 1, 1, d), 64.0))
    change(case, case.v, np.array([32.0, -32.0])[None, None, :, None] * np.ones((1, 1, 2, d)))
    change(case, case.k, np.array([0.1, -0.1])[None, None, :, None] * np.ones((1, 1, 2, d)))
    want = check(case, f"head dim {d}")
    assert 1000 < np.abs(want[0]).max() < 65504
    case.release()


@pytest.mark.parametrize("factor", [2.0 ** -14, 2.0 ** -8, 2.0 ** 8, 2.0 ** 12])
@pytest.mark.parametrize("sq,sk,heads,kv,d", [(70, 70, 2, 2, 64), (150, 300, 4, 2, 128), (40, 600, 2, 1, 40), (70, 90, 2, 1, 256)])
def test_scaled_gradients(gpu, factor, sq, sk, heads, kv, d):
    case = Case(gpu, O.F16, 1, heads, kv, sq, sk, d)
    change(case, case.grad, case.grad.values() * factor)
    change(case, case.k, case.k.values() * 2.0 ** -6)       # (so that large gradients of the scores leave dq and dk within f16)
    change(case, case.q, case.q.values() * 2.0 ** -6)
    check(case, f"gradients times {factor}")
    case.release()


@pytest.mark.parametrize("window,sinks", [(0, 0), (500, 200)])
def test_gradients_that_grow_and_shrink_from_tile_to_tile(gpu, window, sinks):
    """The units of a query's and of a key's sums are set by small values first, then by ones beyond f16, and the other way round."""
    case = Case(gpu, O.F16, 1, 2, 1, 700, 700, 64, causal=False, window=window, sinks=sinks)
    size = 2.0 ** np.linspace(-12, 8, 700)
    rng = np.random.default_rng(9)
    for turn in (1, -1):
        change(case, case.grad, rng.standard_normal((1, 2, 700, 64)) * size[::turn, None])
        change(case, case.v, rng.standard_normal((1, 1, 700, 64)) * size[::turn, None])
        change(case, case.k, rng.standard_normal((1, 1, 700, 64)) * 2.0 ** -7)
        change(case, case.q, rng.standard_normal((1, 2, 700, 64)) * 2.0 ** -7)
        check(case, f"sizes {'rising' if turn == 1 else 'falling'}")
    case.release()


@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 1)])
def test_even_rows_over_many_keys(gpu, heads, kv):
    """Weights of 1 / 20000 are below f16's smallest normal number, and dS further."""
    case = Case(gpu, O.F16, 1, heads, kv, 33, 20000, 64, scale=1e-3)
    change(case, case.grad, case.grad.values() * 2.0 ** -4)
    check(case, "even rows")
    case.release()


def test_zero_gradients_and_rows_that_see_nothing(gpu):
    case = Case(gpu, O.F16, 2, 2, 1, 50, 70, 64, window=20, sinks=2, lengths=[70, 0])
    change(case, case.grad, np.zeros((2, 2, 50, 64)))
    case.forward()
    case.backward()
    gpu.ctx.sync()
    assert all(np.all(b.fetch() == 0) for b in (case.dq, case.dk, case.dv))
    grad = np.zeros((2, 2, 50, 64))
    grad[:, :, 17] = 512.0
    change(case, case.grad, grad)
    check(case, "one gradient")
    case.release()
