"""What the transformer-block operators refuse: every argument is checked before the device is touched, so the checks run
without one (a valid call gets as far as its missing context)."""
import ctypes as C

import pytest

from aix_amd import kernels as K

LIB = K.load()
BASE = 1 << 40            # addresses that nobody reads: the calls end at their checks


class At:
    """Descriptors at addresses apart from one another."""

    def __init__(self):
        self.next = BASE

    def __call__(self, dtype, *shape, strides=None):
        t = K.tensor(self.next, dtype, shape, strides)
        self.next += 1 << 32
        return t


def refused(call, message):
    assert call() == 1
    text = LIB.aixk_last_error().decode()
    assert message in text, text


def attention_parts(backward):
    at = At()
    d = {"q": at(K.BF16, 2, 4, 5, 64), "k": at(K.BF16, 2, 2, 7, 64), "v": at(K.BF16, 2, 2, 7, 64), "out": at(K.BF16, 2, 4, 5, 64), "lse": at(K.F32, 2, 4, 5),
         "lengths": None, "starts": None, "scale": 0.125, "spec": True}
    if backward:
        d.update(grad=at(K.BF16, 2, 4, 5, 64), dq=at(K.BF16, 2, 4, 5, 64), dk=at(K.BF16, 2, 2, 7, 64), dv=at(K.BF16, 2, 2, 7, 64))
    return at, d


def call_attention(d):
    r = lambda t: C.byref(t) if t is not None else None       # noqa: E731
    p = lambda t: C.pointer(t) if t is not None else None      # noqa: E731
    spec = K.AttentionSpec(scale=d["scale"], causal=1, window=3, sinks=1, lengths=p(d["lengths"]), starts=p(d["starts"]))
    s = C.byref(spec) if d["spec"] else None
    if "grad" in d:
        return LIB.aixk_attention_backward(None, r(d["grad"]), r(d["q"]), r(d["k"]), r(d["v"]), r(d["out"]), r(d["lse"]), s, r(d["dq"]), r(d["dk"]), r(d["dv"]))
    return LIB.aixk_attention(None, r(d["q"]), r(d["k"]), r(d["v"]), s, r(d["out"]), r(d["lse"]))


@pytest.mark.parametrize("backward", [False, True])
def test_attention(backward):
    at, good = attention_parts(backward)
    refused(lambda: call_attention(good), "null context")
    cases = [
        ({"q": None}, "bad operand descriptor"),
        ({"spec": False}, "null spec"),
        ({"q": at(K.BF16, 8, 5, 64)}, "must be [batch, heads, sequence, head dim]"),
        ({"k": at(K.F16, 2, 2, 7, 64)}, "one element type"),
        ({"q": at(K.F64, 2, 4, 5, 64)}, "f32, f16 or bf16"),
        ({"v": at(K.BF16, 2, 2, 8, 64)}, "shapes of keys and values differ"),
        ({"q": at(K.BF16, 3, 4, 5, 64)}, "batch or head dim"),
        ({"q": at(K.BF16, 2, 5, 5, 64)}, "a multiple of those of the keys"),
        ({"q": at(K.BF16, 2, 4, 5, 300), "k": at(K.BF16, 2, 2, 7, 300), "v": at(K.BF16, 2, 2, 7, 300)}, "1 .. 256"),
        ({"q": at(K.BF16, 2, 4, 5, 0), "k": at(K.BF16, 2, 2, 7, 0), "v": at(K.BF16, 2, 2, 7, 0)}, "1 .. 256"),
        ({"k": at(K.BF16, 2, 2, 1 << 29, 64, strides=(0, 0, 0, 1)), "v": at(K.BF16, 2, 2, 1 << 29, 64, strides=(0, 0, 0, 1))}, "shorter than 2^29"),
        ({"scale": 0.0}, "positive"), ({"scale": -1.0}, "positive"), ({"scale": float("nan")}, "positive"), ({"scale": float("inf")}, "positive"),
        ({"lengths": at(K.I64, 2)}, "int32 [batch]"), ({"starts": at(K.I32, 3)}, "int32 [batch]"), ({"lengths": at(K.I32, 2, 1)}, "int32 [batch]"),
        ({"lse": at(K.F32, 2, 4, 6)}, "lse"), ({"lse": at(K.BF16, 2, 4, 5)}, "lse"), ({"lse": at(K.F32, 2, 4, 5, strides=(20, 1, 4))}, "dense"),
    ]
    if backward:
        cases += [({"grad": at(K.F16, 2, 4, 5, 64)}, "grad or out"), ({"out": at(K.BF16, 2, 4, 4, 64)}, "shape of the queries"), ({"lse": None}, "lse is needed"),
                  ({"dq": None}, "dq"), ({"dk": at(K.BF16, 2, 2, 5, 64)}, "dk"), ({"dv": at(K.BF16, 2, 2, 7, 64, strides=(0, 448, 64, 1))}, "broadcast"),
                  ({"dq": good["q"]}, "overlaps"), ({"dk": good["v"]}, "overlaps"), ({"dk": good["dv"]}, "share")]
    else:
        cases += [({"out": None}, "the result"), ({"out": at(K.F32, 2, 4, 5, 64)}, "the result"), ({"out": at(K.BF16, 2, 4, 6, 64)}, "does not match"),
                  ({"out": at(K.BF16, 2, 4, 5, 64, strides=(1280, 320, 0, 1))}, "broadcast"), ({"out": good["q"]}, "overlaps"), ({"out": good["v"]}, "does not match"),
                  ({"lse": K.tensor(good["q"].data, K.F32, (2, 4, 5))}, "overlaps"), ({"lse": K.tensor(good["out"].data, K.F32, (2, 4, 5))}, "overlap")]
    wrong = at(K.BF16, 2, 4, 5, 64)
    wrong.size += 1
    cases.append(({"q": wrong}, "size and shape"))
    for change, message in cases:
        refused(lambda: call_attention({**good, **change}), message)
    if not backward:
        refused(lambda: call_attention({**good, "lse": None}), "null context")
