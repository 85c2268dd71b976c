"""Which results of the transformer-block operators may lie in between their operands and one another, and which may not.  The
checks end before the device is touched: a valid call gets as far as its missing context."""
import pytest

from aix_amd import kernels as K

from test_block_operators_refusals import At, attention_parts, call_attention, call_rotary, refused

FINE = "null context"


def packed(at, dtype, batch, length, *heads, d=64, gap=0, order="row"):
    """Views [batch, heads, length, d] side by side in the rows of one projection."""
    base = at(dtype, 1)
    width, views, offset = sum(heads) * d + gap, [], 0
    strides = {"row": (length * width, d, width, 1), "turned": (width, d, batch * width, 1)}[order]
    for h in heads:
        views.append(K.tensor(base.data, dtype, (batch, h, length, d), strides, offset))
        offset += h * d
    return views


def rotary(**parts):
    spec = {"spec": True, "dims": 32, "interleaved": 0, "inverse": 0, "scaling": 0, "base": 1e4, "factor": 1.0, "original_length": 1.0, "low_turns": 0.0, "high_turns": 1.0,
            "magnitude": 1.0}
    return lambda: call_rotary({**spec, **parts})


@pytest.mark.parametrize("order", ["row", "turned"])
@pytest.mark.parametrize("heads", [(4, 4, 4), (8, 2, 2), (1, 1, 1)])
@pytest.mark.parametrize("batch,length", [(2, 5), (1, 5), (3, 1), (1, 1)])
def test_queries_and_keys_of_a_packed_projection_turn_in_place(order, heads, batch, length):
    at = At()
    q, k, v = packed(at, K.BF16, batch, length, *heads, gap=8, order=order)
    positions = at(K.I32, batch, length)
    refused(rotary(q=q, k=k, positions=positions, q_out=q, k_out=k), FINE)
    if heads[0] == heads[2]:
        refused(rotary(q=q, k=k, positions=positions, q_out=v, k_out=k), FINE)
    if heads[1] == heads[2]:
        refused(rotary(q=q, k=k, positions=positions, q_out=q, k_out=v), FINE)


def test_results_in_between_the_operands_of_attention():
    at, good = attention_parts(False)
    q, k, v, out = packed(at, K.BF16, 2, 7, 4, 2, 2, 4)
    refused(lambda: call_attention({**good, "q": q, "k": k, "v": v, "out": out, "lse": at(K.F32, 2, 4, 7)}), FINE)
    refused(lambda: call_attention({**good, "q": q, "k": k, "v": v, "out": q, "lse": at(K.F32, 2, 4, 7)}), "overlaps")
    moved = K.tensor(q.data, K.BF16, (2, 4, 7, 64), list(q.strides[:4]), 8)
    refused(lambda: call_attention({**good, "q": q, "k": k, "v": v, "out": moved, "lse": at(K.F32, 2, 4, 7)}), "overlaps")
    refused(rotary(q=q, k=None, positions=at(K.I32, 2, 7), q_out=moved, k_out=None), "overlaps")


@pytest.mark.parametrize("first,second", [("dq", "dk"), ("dq", "dv"), ("dk", "dv")])
@pytest.mark.parametrize("offset", [0, 1, 64, 300])
def test_gradients_that_share_memory_are_refused(first, second, offset):
    at, good = attention_parts(True)
    shape = tuple(good[second].shape[:4])
    refused(lambda: call_attention({**good, second: K.tensor(good[first].data, K.BF16, shape, None, offset)}), "share")
    refused(lambda: call_attention({**good, first: K.tensor(good[second].data, K.BF16, tuple(good[first].shape[:4]), None, offset)}), "share")


def test_gradients_side_by_side():
    at, good = attention_parts(True)
    dq, dk, dv = packed(at, K.BF16, 2, 7, 4, 2, 2)
    like_q = {n: at(K.BF16, 2, 4, 7, 64) for n in ("q", "grad", "out")}
    refused(lambda: call_attention({**good, **like_q, "lse": at(K.F32, 2, 4, 7), "dq": dq, "dk": dk, "dv": dv}), FINE)
    dv.offset += 4
    refused(lambda: call_attention({**good, **like_q, "lse": at(K.F32, 2, 4, 7), "dq": dq, "dk": dk, "dv": dv}), "share")     # (its last elements: the next row's first)


@pytest.mark.parametrize("offset", [0, 1, 64])
def test_turned_queries_and_keys_that_share_memory_are_refused(offset):
    at = At()
    q, k, positions, q_out = at(K.F32, 2, 4, 5, 64), at(K.F32, 2, 2, 5, 64), at(K.I32, 2, 5), at(K.F32, 2, 4, 5, 64)
    refused(rotary(q=q, k=k, positions=positions, q_out=q_out, k_out=K.tensor(q_out.data, K.F32, (2, 2, 5, 64), None, offset)), "share")


@pytest.mark.parametrize("strides", [(1280, 320, 1, 1), (1280, 63, 252, 1), (64, 1280, 64, 1), (1280, 320, 64, 2), (1280, 64, 200, 1)])
def test_results_that_meet_an_element_twice_are_refused(strides):
    at, good = attention_parts(False)
    refused(lambda: call_attention({**good, "out": at(K.BF16, 2, 4, 5, 64, strides=strides)}), "twice")
    at, good = attention_parts(True)
    for name in ("dq", "dk", "dv"):
        refused(lambda: call_attention({**good, name: at(K.BF16, *good[name].shape[:4], strides=strides)}), "twice")
    q, k, positions = at(K.F32, 2, 4, 5, 64), at(K.F32, 2, 4, 5, 64), at(K.I32, 2, 5)
    refused(rotary(q=q, k=k, positions=positions, q_out=at(K.F32, 2, 4, 5, 64, strides=strides), k_out=k), "twice")
    refused(rotary(q=q, k=k, positions=positions, q_out=q, k_out=at(K.F32, 2, 4, 5, 64, strides=strides)), "twice")


@pytest.mark.parametrize("shape,strides", [((2, 4, 5, 64), (1280, 64, 256, 1)), ((2, 4, 5, 64), (1, 2, 512, 8)), ((2, 4, 5, 64), (10 ** 6, 10 ** 5, 10 ** 4, 3)),
                                           ((1, 4, 5, 64), (0, 320, 64, 1)), ((2, 4, 1, 64), (256, 64, 1, 1)), ((2, 4, 5, 1), (20, 5, 1, 0))])
def test_results_of_any_order(shape, strides):
    at = At()
    q = at(K.BF16, *shape)
    refused(rotary(q=q, k=None, positions=at(K.I32, shape[0], shape[2]), q_out=at(K.BF16, *shape, strides=strides), k_out=None, dims=2 if shape[3] > 1 else 0),
            FINE if shape[3] > 1 else "turned part")
    k = at(K.BF16, shape[0], shape[1], 7, shape[3])
    parts = {"q": q, "k": k, "v": at(K.BF16, *k.shape[:4]), "out": at(K.BF16, *shape, strides=strides), "lse": None, "lengths": None, "starts": None, "scale": 1.0, "spec": True}
    refused(lambda: call_attention(parts), FINE)


def cells(t):
    """The element positions of a view."""
    got = [int(t.offset)]
    for d in range(t.rank):
        got = [p + n * int(t.strides[d]) for p in got for n in range(int(t.shape[d]))]
    return got


def test_whatever_shares_an_element_is_refused():
    """Random views of one piece of memory: a call with a result and an operand that share an element is never let through."""
    import random
    rng, at, apart = random.Random(5), At(), 0
    positions = at(K.I32, 2, 3)
    base = at(K.F32, 1)
    for _ in range(4000):
        views = []
        for _ in range(2):
            dims, strides, run = rng.sample(range(4), 4), [0] * 4, 1
            shape = (2, 2, 3, 4)
            for d in dims:
                strides[d], run = run, run * shape[d] * rng.choice((1, 1, 1, 2, 3)) + rng.choice((0, 0, 4, 8))
            views.append(K.tensor(base.data, K.F32, shape, strides, rng.choice((0, 4, 8, 16, rng.randrange(64)))))
        q, out = views
        first, second = set(cells(q)), cells(out)
        assert rotary(q=q, k=None, positions=positions, q_out=out, k_out=None, dims=4)() == 1
        text = K.load().aixk_last_error().decode()
        same = q.offset == out.offset and list(q.strides[:4]) == list(out.strides[:4])
        if same or "overlaps" not in text:
            assert same or not first & set(second), (list(q.strides[:4]), q.offset, list(out.strides[:4]), out.offset)
            assert FINE in text
            apart += not same
    assert apart                                             # (the rule lets some through: those that it can show to be apart)
