"""A query that holds a NaN gives a row of NaNs whichever kernel takes it, never the zeros of a query that sees no key, and leaves the
other rows as they are.  Bounds: blockref.py."""
import numpy as np
import pytest

import blockref as R
import gpuharness as G
from oracle import cpuref as O

from test_gpu_attention import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    g = G.Gpu()
    yield g
    g.close()


@pytest.mark.parametrize("dtype", [O.BF16, O.F16, O.F32])
@pytest.mark.parametrize("sq,sk,d,window", [(1, 40, 64, 0), (1, 600, 64, 0), (1, 20000, 128, 0), (3, 9000, 256, 700), (40, 3000, 128, 0), (130, 130, 64, 0), (300, 300, 200, 50)])
def test_a_nan_query(gpu, dtype, sq, sk, d, window):
    case = Case(gpu, dtype, 2, 4, 2, sq, sk, d, window=window, sinks=1, lengths=[sk, 0])
    store = case.q.before.copy()
    bad = (0, 1, sq // 2)
    case.q.view(store)[bad + (d // 3,)] = R.T_round(np.float32(np.nan), dtype)
    gpu.ctx.upload(case.q.ptr, store)
    case.forward()
    gpu.ctx.sync()
    out, lse, out_far, lse_far = R.attention(case.q.values(), case.k.values(), case.v.values(), case.seen, case.scale, dtype)
    got, stat = case.out.fetch(), case.lse.fetch()
    assert np.all(np.isnan(got[bad])) and np.isnan(stat[bad])
    got[bad], stat[bad] = out[bad], lse[bad]
    assert np.array_equal(np.isneginf(stat), np.isneginf(lse))
    R.check(stat, lse, lse_far, "lse")
    R.check(got, out, out_far, "out")
    case.release()
