"""Sizes on both sides of the choice between workgroups of queries and shares of the keys, for every type and padded head dim.
Bounds: blockref.py."""
import pytest

import gpuharness as G
from oracle import cpuref as O

from test_gpu_attention import Case, both_ways

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    g = G.Gpu()
    yield g
    g.close()


@pytest.mark.parametrize("dtype", [O.BF16, O.F16, O.F32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("batch,heads,kv,sq,sk", [(1, 4, 4, 256, 256), (1, 4, 4, 512, 512), (1, 8, 2, 130, 1500), (2, 12, 12, 40, 512), (3, 2, 2, 700, 700), (1, 2, 1, 900, 2500)])
def test_both_sides(gpu, dtype, d, batch, heads, kv, sq, sk):
    both_ways(Case(gpu, dtype, batch, heads, kv, sq, sk, d, lengths=[sk, sk // 3, 5][:batch]), f"{sq} x {sk}", backward=False)
