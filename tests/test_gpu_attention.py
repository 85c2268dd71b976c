"""aixk_attention and aixk_attention_backward against plain 64-bit implementations, at the sizes, masks and layouts where
they can go wrong.  Tolerances are the rounding bounds of blockref.py."""
import ctypes as C
import math

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


BHSD, BSHD = (0, 1, 2, 3), (0, 2, 1, 3)


class Case:
    def __init__(self, gpu, dtype, batch, heads, kv, sq, sk, d, causal=True, window=0, sinks=0, lengths=None, starts=None, order=BSHD,
                 pad=0, seed=0, scale=None, offset=0, spread=1.0):
        rng = np.random.default_rng(seed + 1000 * sq + sk + d)
        self.gpu, self.dtype = gpu, dtype
        self.scale = d ** -0.5 if scale is None else scale
        make = lambda h, s: rng.standard_normal((batch, h, s, d)) * spread                # noqa: E731
        box = lambda shape, values=None, fill=None: R.Box(gpu, K, dtype, shape, values, order, pad, offset, fill)      # noqa: E731
        self.q, self.k, self.v = box((batch, heads, sq, d), make(heads, sq)), box((batch, kv, sk, d), make(kv, sk)), box((batch, kv, sk, d), make(kv, sk))
        self.grad = box((batch, heads, sq, d), make(heads, sq))
        self.out = box((batch, heads, sq, d), fill=7.0)
        self.lse = R.Box(gpu, K, O.F32, (batch, heads, sq), fill=7.0)
        self.dq, self.dk, self.dv = box((batch, heads, sq, d), fill=7.0), box((batch, kv, sk, d), fill=7.0), box((batch, kv, sk, d), fill=7.0)
        self.kept = []
        self.lengths, self.starts = lengths, starts
        self.spec = K.AttentionSpec(scale=self.scale, causal=int(causal), window=window, sinks=sinks, lengths=self.ints(lengths), starts=self.ints(starts))
        self.scale = float(np.float32(self.scale))
        self.seen = R.visible(batch, sq, sk, causal, window, sinks, lengths, starts)

    def ints(self, values):
        if values is None:
            return None
        box = R.Box(self.gpu, K, O.I32, (len(values),), np.asarray(values, np.float64))
        self.kept.append(box)
        return C.pointer(box.desc)

    def forward(self, lse=True):
        G.run_gpu(self.gpu, "aixk_attention", G.ref(self.q.desc), G.ref(self.k.desc), G.ref(self.v.desc), C.byref(self.spec), G.ref(self.out.desc),
                  G.ref(self.lse.desc) if lse else None)

    def backward(self):
        G.run_gpu(self.gpu, "aixk_attention_backward", G.ref(self.grad.desc), G.ref(self.q.desc), G.ref(self.k.desc), G.ref(self.v.desc), G.ref(self.out.desc),
                  G.ref(self.lse.desc), C.byref(self.spec), G.ref(self.dq.desc), G.ref(self.dk.desc), G.ref(self.dv.desc))

    def check_forward(self, what):
        out, lse, out_far, lse_far = R.attention(self.q.values(), self.k.values(), self.v.values(), self.seen, self.scale, self.dtype)
        got = self.lse.fetch()
        assert np.array_equal(np.isneginf(got), np.isneginf(lse)), f"{what}: rows without a visible key"
        R.check(got, lse, lse_far, what + " lse")
        R.check(self.out.fetch(), out, out_far, what + " out")

    def check_backward(self, what):
        self.gpu.ctx.sync()
        got, far = R.attention_backward(self.grad.values(), self.q.values(), self.k.values(), self.v.values(), self.out.fetch(), self.lse.fetch(), self.seen,
                                        self.scale, self.dtype)
        for box, want, f, name in zip((self.dq, self.dk, self.dv), got, far, ("dq", "dk", "dv")):
            R.check(box.fetch(), want, f, f"{what} {name}")

    def release(self):
        self.gpu.release()


def both_ways(case, what, backward=True):
    case.forward()
    case.check_forward(what)
    if backward:
        case.backward()
        case.check_backward(what)
    case.release()


DTYPES = [O.BF16, O.F16, O.F32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256, 8, 40, 33, 1, 200])
def test_head_dims(gpu, dtype, d):
    both_ways(Case(gpu, dtype, 1, 2, 2, 70, 70, d), f"head dim {d}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq,sk", [(1, 1), (2, 3), (1, 300), (31, 33), (129, 129), (64, 257), (200, 70), (17, 1000)])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(gpu, dtype, sq, sk, causal):
    both_ways(Case(gpu, dtype, 2, 4, 2, sq, sk, 64, causal=causal), f"{sq} queries on {sk} keys, causal {causal}")


@pytest.mark.parametrize("dtype", [O.BF16, O.F32])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (64, 4), (65, 64), (100, 70), (1000, 3), (1 << 40, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_windows_and_leading_keys(gpu, dtype, window, sinks, causal):
    both_ways(Case(gpu, dtype, 1, 2, 1, 300, 300, 64, causal=causal, window=window, sinks=sinks), f"window {window}, {sinks} leading keys")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal,window,sinks,heads,kv", [(True, 40, 4, 2, 2), (False, 40, 4, 2, 1), (True, 64, 140, 4, 2), (False, 30, 300, 2, 2), (True, 200, 129, 3, 1)])
def test_leading_keys_far_from_their_queries(gpu, dtype, causal, window, sinks, heads, kv):
    """Queries that see nothing but the leading keys have workgroups of their own in the backward pass."""
    both_ways(Case(gpu, dtype, 2, heads, kv, 700, 700, 64, causal=causal, window=window, sinks=sinks, lengths=[700, 150]), f"window {window}, {sinks} leading keys")
    both_ways(Case(gpu, dtype, 2, heads, kv, 650, 700, 64, causal=causal, window=window, sinks=sinks, lengths=[700, 3], starts=[20, 600]), f"window {window}, {sinks} leading keys, later")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,heads,kv", [(5, 8, 4), (9, 16, 16)])
@pytest.mark.parametrize("sq,sk,d", [(200, 200, 64), (130, 200, 40), (150, 150, 128), (129, 161, 192)])
def test_many_rows(gpu, dtype, batch, heads, kv, sq, sk, d):
    """Enough rows for workgroups of 64 queries, and of 128."""
    lengths = [sk, 0, 1, sk - 1, sk // 2, 10 ** 6, -1, 65, 33][:batch]
    for causal, window, sinks in ((True, 0, 0), (False, 0, 0), (True, 30, 3), (False, 70, 66)):
        both_ways(Case(gpu, dtype, batch, heads, kv, sq, sk, d, causal=causal, window=window, sinks=sinks, lengths=lengths), f"causal {causal}, window {window}")
    both_ways(Case(gpu, dtype, batch, heads, kv, sq, sk, d, window=50, sinks=2, lengths=lengths, starts=[5, 0, -3, 70, 2 ** 31 - 1, -2 ** 31, sk - 1, 0, 40][:batch]), "starts")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,sq,d", [(8, 2, 64, 64), (4, 4, 50, 128), (6, 2, 33, 80), (2, 2, 100, 192), (4, 1, 17, 256)])
def test_some_queries_far_into_a_cache(gpu, dtype, heads, kv, sq, d):
    """The next part of a prompt: the keys of its rows in shares."""
    for window, sinks in ((0, 0), (300, 4)):
        both_ways(Case(gpu, dtype, 2, heads, kv, sq, 3000, d, window=window, sinks=sinks, lengths=[3000, 1234]), f"{sq} queries, window {window}")


@pytest.mark.parametrize("dtype", [O.BF16, O.F16])
@pytest.mark.parametrize("sq", [1, 3, 40, 150])
@pytest.mark.parametrize("causal,window,sinks", [(True, 0, 0), (True, 20, 3), (False, 20, 3), (False, 0, 0)])
def test_every_sequence_its_own_length(gpu, dtype, sq, causal, window, sinks):
    lengths = [150, 0, 1, 77, 149, -5, 10 ** 6]
    both_ways(Case(gpu, dtype, 7, 6, 2, sq, 150, 64, causal=causal, window=window, sinks=sinks, lengths=lengths), f"{sq} queries, lengths")
    both_ways(Case(gpu, dtype, 7, 6, 2, sq, 150, 64, causal=causal, window=window, sinks=sinks, lengths=lengths, starts=[0] * 7), f"{sq} queries, lengths from the left")
    both_ways(Case(gpu, dtype, 7, 3, 3, sq, 150, 32, causal=causal, window=window, sinks=sinks, lengths=lengths, starts=[5, 0, -3, 70, 2 ** 31 - 1, -2 ** 31, 149]),
              f"{sq} queries, lengths and starts")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv", [(8, 1), (12, 4), (5, 5), (32, 2)])
@pytest.mark.parametrize("sq", [1, 2, 90])
def test_shared_key_heads(gpu, dtype, heads, kv, sq):
    both_ways(Case(gpu, dtype, 2, heads, kv, sq, 90, 64, window=50, sinks=2), f"{heads} heads on {kv}, {sq} queries")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [2, 75])
@pytest.mark.parametrize("order,pad,offset,d", [(BHSD, 0, 0, 64), (BSHD, 8, 0, 64), (BSHD, 3, 5, 64), ((0, 1, 3, 2), 0, 0, 64), ((3, 0, 1, 2), 0, 1, 40), ((2, 0, 1, 3), 0, 16, 72)])
def test_layouts(gpu, dtype, sq, order, pad, offset, d):
    both_ways(Case(gpu, dtype, 2, 4, 2, sq, 75, d, order=order, pad=pad, offset=offset, window=30, sinks=1), f"order {order}, pad {pad}, offset {offset}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sq", [1, 50])
def test_large_scores_and_scales(gpu, dtype, sq):
    both_ways(Case(gpu, dtype, 1, 2, 2, sq, 300, 64, scale=1.0, spread=2.0), "scores of some tens")
    both_ways(Case(gpu, dtype, 1, 2, 2, sq, 300, 64, scale=1e-6), "an almost even mean")


@pytest.mark.parametrize("sq", [1, 5, 64])
def test_nothing_behind_a_length_is_read(gpu, sq):
    """Cache rows that were never written may hold anything."""
    for bad in (np.nan, np.inf, -3.0e38):
        case = Case(gpu, O.BF16, 2, 4, 2, sq, 200, 64, lengths=[70, 131])
        for box in (case.k, case.v):
            store = box.before.copy()
            view = box.view(store)
            view[0, :, 70:], view[1, :, 131:] = R.T_round(np.float32(bad), O.BF16), R.T_round(np.float32(bad), O.BF16)
            gpu.ctx.upload(box.ptr, store)
        case.forward()
        case.check_forward(f"{bad} behind the length")
        case.backward()
        case.gpu.ctx.sync()
        want, far = R.attention_backward(case.grad.values(), case.q.values(), case.k.values(), case.v.values(), case.out.fetch(), case.lse.fetch(), case.seen, case.scale, O.BF16)
        R.check(case.dq.fetch(), want[0], far[0], "dq")
        R.check(case.dk.fetch(), want[1], far[1], "dk")
        R.check(case.dv.fetch(), want[2], far[2], "dv")
        case.release()


@pytest.mark.parametrize("keys", [4096, 20000])
@pytest.mark.parametrize("window", [0, 777])
def test_long_caches_are_split_and_joined(gpu, keys, window):
    case = Case(gpu, O.BF16, 2, 4, 1, 1, keys, 128, window=window, sinks=5, lengths=[keys, keys // 3])
    both_ways(case, f"{keys} keys, window {window}", backward=False)


def test_without_lse(gpu):
    case = Case(gpu, O.F16, 1, 2, 1, 40, 40, 64)
    case.forward(lse=False)
    assert np.all(case.lse.fetch() == 7.0)
    out, _, far, _ = R.attention(case.q.values(), case.k.values(), case.v.values(), case.seen, case.scale, O.F16)
    R.check(case.out.fetch(), out, far, "out")
    case.release()


@pytest.mark.parametrize("shape", [(0, 2, 2, 5, 5), (1, 2, 2, 0, 5), (1, 2, 2, 5, 0), (1, 4, 2, 1, 0), (2, 0, 0, 3, 3)])
def test_empty_sizes(gpu, shape):
    b, h, kv, sq, sk = shape
    case = Case(gpu, O.BF16, b, h, kv, sq, sk, 64)
    case.forward()
    case.backward()
    gpu.ctx.sync()
    if case.out.count and sk == 0:
        assert np.all(case.out.fetch() == 0) and np.all(np.isneginf(case.lse.fetch())) and np.all(case.dq.fetch() == 0)
    if sq == 0 and b and h:
        assert np.all(case.dk.fetch() == 0) and np.all(case.dv.fetch() == 0)
    case.release()


@pytest.mark.parametrize("sq", [1, 130])
def test_repeats_bit_for_bit(gpu, sq):
    case = Case(gpu, O.BF16, 2, 8, 2, sq, 500, 64)
    results = []
    for _ in range(3):
        case.forward()
        case.backward()
        results.append([b.fetch().tobytes() for b in (case.out, case.lse, case.dq, case.dk, case.dv)])
    assert results[0] == results[1] == results[2]
    case.release()


def test_gradients_against_differences(gpu):
    """f32: the directional derivative of sum(out w) along a random direction, by a central difference of the kernel's own
    forward pass.  The difference of step 2^-6 is off by the third derivative (about step^2) and by the rounding of the two
    sums (2^-24 of their mass over the step): 2 % of the gradient's length covers both."""
    case = Case(gpu, O.F32, 1, 2, 1, 20, 20, 16, window=9, sinks=2)
    case.forward()
    case.backward()
    w = case.grad.values()
    rng = np.random.default_rng(5)
    for box, grad in ((case.q, case.dq), (case.k, case.dk), (case.v, case.dv)):
        way = rng.standard_normal(box.shape)
        way /= np.sqrt((way ** 2).sum())
        step, sums = 2.0 ** -6, []
        for sign in (1, -1):
            store = box.before.copy()
            box.view(store)[...] = (box.values() + sign * step * way).astype(np.float32)
            gpu.ctx.upload(box.ptr, store)
            case.forward()
            sums.append((case.out.fetch() * w).sum())
        gpu.ctx.upload(box.ptr, box.before)
        g = grad.fetch()
        assert abs((sums[0] - sums[1]) / (2 * step) - (g * way).sum()) <= 0.02 * np.sqrt((g ** 2).sum())
    case.release()
