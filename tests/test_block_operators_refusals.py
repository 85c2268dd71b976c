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


def ref(t):
    return C.byref(t) if t is not None else None


def ptr(t):
    return C.pointer(t) if t is not None else None


def call_rotary(d):
    spec = K.RotarySpec(**{n: d[n] for n, _ in K.RotarySpec._fields_})
    return LIB.aixk_rotary(None, ref(d["q"]), ref(d["k"]), ref(d["positions"]), C.byref(spec) if d["spec"] else None, ref(d["q_out"]), ref(d["k_out"]))


def test_rotary():
    at = At()
    good = {"q": at(K.F16, 2, 4, 5, 64), "k": at(K.F16, 2, 1, 5, 64), "positions": at(K.I32, 2, 5), "q_out": at(K.F16, 2, 4, 5, 64), "k_out": at(K.F16, 2, 1, 5, 64),
            "spec": True, "dims": 32, "interleaved": 0, "inverse": 0, "scaling": K.ROTARY_PARTS, "base": 1e4, "factor": 4.0, "original_length": 4096.0, "low_turns": 1.0,
            "high_turns": 32.0, "magnitude": 1.0}
    refused(lambda: call_rotary(good), "null context")
    refused(lambda: call_rotary({**good, "k": None, "k_out": None}), "null context")
    refused(lambda: call_rotary({**good, "q_out": good["q"], "k_out": good["k"]}), "null context")          # in place
    nan, inf = float("nan"), float("inf")
    for change, message in [
        ({"spec": False}, "null spec"), ({"q": None}, "the queries"), ({"k": None}, "belong together"), ({"k_out": None}, "belong together"),
        ({"q": at(K.F16, 4, 5, 64)}, "[batch, heads, sequence, head dim]"), ({"q": at(K.F64, 2, 4, 5, 64)}, "f32, f16 or bf16"),
        ({"q_out": at(K.BF16, 2, 4, 5, 64)}, "bad descriptor"), ({"q_out": at(K.F16, 2, 5, 4, 64)}, "differs"), ({"k_out": at(K.F16, 2, 1, 5, 64, strides=(0, 0, 64, 1))}, "broadcast"),
        ({"k": at(K.BF16, 2, 1, 5, 64), "k_out": at(K.BF16, 2, 1, 5, 64)}, "differ in type"), ({"k": at(K.F16, 2, 1, 6, 64), "k_out": at(K.F16, 2, 1, 6, 64)}, "sequence"),
        ({"positions": None}, "int32"), ({"positions": at(K.I64, 2, 5)}, "int32"), ({"positions": at(K.I32, 5)}, "int32"), ({"positions": at(K.I32, 5, 2)}, "int32"),
        ({"dims": 0}, "turned part"), ({"dims": 31}, "turned part"), ({"dims": 66}, "turned part"), ({"base": 0.0}, "positive"), ({"base": nan}, "positive"),
        ({"magnitude": 0.0}, "positive"), ({"scaling": 4}, "unknown scaling"), ({"scaling": -1}, "unknown scaling"), ({"factor": 0.0}, "factor"), ({"factor": inf}, "factor"),
        ({"original_length": 0.0}, "original length"), ({"low_turns": 32.0}, "high_turns"),
        ({"q_out": good["k"]}, "bad descriptor"), ({"k_out": K.tensor(good["q"].data, K.F16, (2, 1, 5, 64))}, "overlaps"),
        ({"q_out": K.tensor(good["q"].data, K.F16, (2, 4, 5, 64), offset=64)}, "overlaps"), ({"k_out": K.tensor(good["q_out"].data, K.F16, (2, 1, 5, 64))}, "share"),
    ]:
        refused(lambda: call_rotary({**good, **change}), message)


def test_matmul_epilogue():
    at = At()
    good = {"a": at(K.BF16, 6, 8), "b": at(K.BF16, 8, 10), "bias": at(K.BF16, 10), "residual": at(K.BF16, 6, 10), "pre": at(K.BF16, 6, 10), "out": at(K.BF16, 6, 10), "act": 2, "spec": True}

    def call(d):
        spec = K.Epilogue(bias=ptr(d["bias"]), residual=ptr(d["residual"]), pre=ptr(d["pre"]), activation=d["act"])
        return LIB.aixk_matmul_epilogue(None, ref(d["a"]), ref(d["b"]), C.byref(spec) if d["spec"] else None, ref(d["out"]))

    for fine in ({}, {"bias": None, "residual": None, "pre": None}, {"bias": at(K.BF16, 1, 10)}, {"out": good["residual"]}, {"residual": at(K.BF16, 6, 10, strides=(0, 1))}):
        refused(lambda: call({**good, **fine}), "null context")
    for change, message in [
        ({"spec": False}, "null epilogue"), ({"a": None}, "2-D"), ({"a": at(K.BF16, 1, 6, 8)}, "2-D"), ({"b": at(K.BF16, 9, 10)}, "inner dimensions"),
        ({"b": at(K.F16, 8, 10)}, "one element type"), ({"a": at(K.I32, 6, 8), "b": at(K.I32, 8, 10)}, "one element type"), ({"a": at(K.F64, 6, 8), "b": at(K.F64, 8, 10)}, "one element type"),
        ({"out": None}, "the result"), ({"out": at(K.F32, 6, 10)}, "the result"), ({"out": at(K.BF16, 6, 10, strides=(12, 1))}, "the result"), ({"out": at(K.BF16, 10, 6)}, "the result"),
        ({"bias": at(K.F32, 10)}, "bias"), ({"bias": at(K.BF16, 6)}, "bias"), ({"bias": at(K.BF16, 10, 1)}, "bias"), ({"residual": at(K.BF16, 10)}, "residual"),
        ({"pre": at(K.BF16, 6, 10, strides=(1, 6))}, "pre"), ({"act": 4}, "unknown activation"), ({"act": -1}, "unknown activation"),
        ({"out": K.tensor(good["a"].data, K.BF16, (6, 10))}, "overlaps an operand"), ({"pre": good["out"]}, "pre overlaps"), ({"pre": good["residual"]}, "pre overlaps"),
        ({"residual": K.tensor(good["out"].data, K.BF16, (6, 10), (0, 1))}, "overlaps the residual"), ({"bias": K.tensor(good["out"].data, K.BF16, (10,))}, "overlaps an operand"),
    ]:
        refused(lambda: call({**good, **change}), message)


def test_matmul_epilogue_backward():
    at = At()
    good = {"grad": at(K.F32, 6, 10), "a": at(K.F32, 6, 8), "b": at(K.F32, 8, 10), "pre": at(K.F32, 6, 10), "act": 3, "dz": at(K.F32, 6, 10), "da": at(K.F32, 6, 8),
            "db": at(K.F32, 8, 10), "dbias": at(K.F32, 10)}

    def call(d):
        return LIB.aixk_matmul_epilogue_backward(None, ref(d["grad"]), ref(d["a"]), ref(d["b"]), ref(d["pre"]), d["act"], ref(d["dz"]), ref(d["da"]), ref(d["db"]), ref(d["dbias"]))

    for fine in ({}, {"da": None, "db": None, "dbias": None}, {"act": 0, "pre": None, "dz": None}, {"dbias": at(K.F32, 1, 10)}):
        refused(lambda: call({**good, **fine}), "null context")
    for change, message in [
        ({"grad": None}, "grad"), ({"grad": at(K.F32, 10, 6)}, "grad"), ({"pre": None}, "needs pre and dz"), ({"dz": None}, "needs pre and dz"), ({"pre": at(K.F16, 6, 10)}, "pre"),
        ({"dz": at(K.F32, 6, 10, strides=(1, 6))}, "dz"), ({"da": at(K.F32, 6, 10)}, "da"), ({"db": at(K.F32, 10, 8)}, "db"), ({"dbias": at(K.F32, 8)}, "dbias"),
        ({"b": at(K.F32, 7, 10)}, "inner dimensions"), ({"act": 9}, "unknown activation"), ({"dz": good["grad"]}, "overlaps an operand"), ({"da": good["a"]}, "overlaps an operand"),
        ({"dbias": K.tensor(good["dz"].data, K.F32, (10,))}, "results overlap"),
    ]:
        refused(lambda: call({**good, **change}), message)
