"""The transformer-block operators as they are used: attention with a sliding window and leading keys that stay
visible (forward, backward, and single tokens over a cache), rotary positions of queries and keys, and the matrix
product with bias, activation and residual in its epilogue (forward and backward).

A case is a dict of plain values; prepare() makes its tensors, run() is one call -- in elementary torch operations
where `own` is false, through the kernel layer (aix_amd.kernels, include/aixhip_kernels.h) where it is true -- and
exact() is the operator's definition in 64 bits.

The kernel layer's calls run on a stream of their context, which does not wait for torch's nor torch's for it: prepare() ends
with its inputs complete, and a program waits for the device (torch.cuda.synchronize()) before it reads the results of
run() or drops a state that a run() still uses."""
import ctypes
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
ACTIVATIONS = ("none", "relu", "gelu", "silu")
SCALINGS = ("plain", "linear", "base", "parts")


def listed():
    def attention(name, op, dtype, batch, heads, kv_heads, q_len, k_len, dim, window, sinks, ragged, causal=True):
        return {"name": name, "op": op, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "q_len": q_len,
                "k_len": k_len, "dim": dim, "window": window, "sinks": sinks, "ragged": ragged, "causal": causal}

    def rotary(name, dtype, batch, heads, kv_heads, length, dim, rotated, interleaved, scaling, far, inverse):
        return {"name": name, "op": "rotary", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "length": length,
                "dim": dim, "rotated": rotated, "interleaved": interleaved, "scaling": scaling, "far": far, "inverse": inverse}

    def product(name, op, dtype, rows, inner, columns, activation, residual, keep, transposed):
        return {"name": name, "op": op, "dtype": dtype, "rows": rows, "inner": inner, "columns": columns,
                "activation": activation, "residual": residual, "keep": keep, "transposed": transposed}

    return [
        # one new token of one short conversation in the 12-head, 64-wide model of the benchmark: nothing but latency
        attention("decode one", "attention", "bf16", 1, 12, 12, 1, 512, 64, 0, 0, False),
        # a full serving batch over a long cache, every sequence at a length of its own: reading the cache is all there is
        attention("decode batch", "attention", "bf16", 16, 32, 8, 1, 32768, 128, 0, 0, True),
        # the same with a window: of the long cache only its end and the first tokens are read
        attention("decode window", "attention", "f16", 32, 32, 4, 1, 16384, 128, 2048, 4, True),
        # a long prompt taken in at once
        attention("prompt", "attention", "bf16", 1, 32, 8, 8192, 8192, 128, 2048, 4, False),
        # odd everything: a padded batch in 32 bits, heads of 80, one sequence empty
        attention("padded f32", "attention", "f32", 4, 6, 2, 777, 777, 80, 200, 3, True),
        # a training step of the benchmark's transformer: 16 sequences of 512, 12 heads of 64
        attention("train backward", "attention_backward", "bf16", 16, 12, 12, 512, 512, 64, 128, 4, False),
        # a training step on a long text with shared key heads
        attention("long backward", "attention_backward", "bf16", 1, 16, 4, 4096, 4096, 128, 1024, 4, False),
        # the new tokens of a serving batch, far into their texts
        rotary("rotary step", "bf16", 8, 32, 8, 1, 128, 128, False, "parts", 120000, False),
        # the gradient on its way back through the positions of a training batch, a part of every head rotated
        rotary("rotary train", "f16", 16, 16, 16, 2048, 128, 64, True, "plain", 0, True),
        # a feed-forward layer for seven tokens: reading the weights is all there is
        product("product few rows", "product", "bf16", 7, 768, 2048, "gelu", False, False, False),
        # a feed-forward layer of a training batch: activation, residual, and what the backward pass needs
        product("product large", "product", "bf16", 8192, 4096, 4096, "gelu", True, True, False),
        # its backward pass at the benchmark's width
        product("product backward", "product_backward", "bf16", 8192, 768, 768, "gelu", False, False, False),
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is spread evenly."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("attention", "attention", "decode", "attention_backward", "attention_backward", "rotary", "product", "product", "product_backward"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op in ("attention", "decode", "attention_backward"):
        kv_heads, group = rng.choice((1, 2, 3, 4, 8, 12)), rng.choice((1, 1, 2, 3, 4, 8))
        dim = rng.choice((32, 40, 64, 64, 72, 80, 96, 128, 128, 192, 256, 33))
        batch = _spread(rng, 1, 16)
        if op == "decode":
            q_len, k_len = rng.choice((1, 1, 1, 2, 5, 16)), _spread(rng, 1, 32768)
            while batch * kv_heads * k_len * dim > 1 << 29:
                k_len = k_len // 2 + 1
        else:
            k_len = _spread(rng, 1, 8192)
            most = 1 << (27 if op == "attention_backward" else 30)
            while batch * kv_heads * group * k_len * k_len > most:
                k_len = k_len * 2 // 3
            q_len = k_len
        window = rng.choice((0, _spread(rng, 1, 4096), _spread(rng, 16, 1024)))
        return {"op": "attention_backward" if op == "attention_backward" else "attention", "dtype": dtype, "batch": batch,
                "heads": kv_heads * group, "kv_heads": kv_heads, "q_len": q_len, "k_len": k_len, "dim": dim, "window": window,
                "sinks": rng.choice((0, 1, 4, 70)) if window else 0, "ragged": rng.random() < 0.5, "causal": rng.random() < 0.8}
    if op == "rotary":
        kv_heads = rng.choice((1, 2, 4, 8))
        dim = rng.choice((32, 64, 80, 96, 128, 256))
        batch, length = _spread(rng, 1, 32), _spread(rng, 1, 8192)
        while batch * length * kv_heads * 5 * dim > 1 << 28:
            length = length // 2 + 1
        return {"op": "rotary", "dtype": dtype, "batch": batch, "heads": kv_heads * rng.choice((1, 2, 4)), "kv_heads": kv_heads, "length": length,
                "dim": dim, "rotated": rng.choice((dim, dim, dim // 2, dim // 4 // 2 * 2)), "interleaved": rng.random() < 0.5, "scaling": rng.choice(SCALINGS),
                "far": rng.choice((0, 0, 5000, 1000000)), "inverse": rng.random() < 0.5}
    rows, inner, columns = _spread(rng, 1, 16384), _spread(rng, 16, 8192), _spread(rng, 16, 8192)
    if rng.random() < 0.7:                                  # widths of models are whole multiples; the others are odd ones
        inner, columns = (inner + 63) // 64 * 64, (columns + 63) // 64 * 64
    while rows * inner * columns > (1 << 35 if dtype != "f32" else 1 << 33):
        rows = rows // 2 + 1
    return {"op": op, "dtype": dtype, "rows": rows, "inner": inner, "columns": columns, "activation": rng.choice(ACTIVATIONS[1:] if op == "product_backward" else ACTIVATIONS),
            "residual": op == "product" and rng.random() < 0.5, "keep": op == "product" and rng.random() < 0.5, "transposed": rng.random() < 0.4}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _heads(g, c, heads, length):
    """[batch, heads, length, dim] as projections leave it: a view of [batch, length, heads, dim]."""
    x = torch.randn((c["batch"], length, heads, c["dim"]), generator=g, device="cuda", dtype=torch.float32)
    return x.to(DTYPES[c["dtype"]]).transpose(1, 2)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c, dt = case, DTYPES[case["dtype"]]
    s = {"case": c}
    if c["op"] in ("attention", "attention_backward"):
        s["q"] = _heads(g, c, c["heads"], c["q_len"])
        s["k"], s["v"] = _heads(g, c, c["kv_heads"], c["k_len"]), _heads(g, c, c["kv_heads"], c["k_len"])
        s["lengths"] = s["starts"] = None
        if c["ragged"]:                                     # serving and padded batches: every sequence its own length, one may be empty
            u = torch.rand((c["batch"],), generator=g, device="cuda")
            lengths = (u * (c["k_len"] + 1)).to(torch.int32).clamp_(max=c["k_len"])
            if c["batch"] > 2:
                lengths[1] = 0
            s["lengths"] = lengths
            if c["q_len"] == c["k_len"]:                    # padded on the right: query i stands at position i
                s["starts"] = torch.zeros((c["batch"],), dtype=torch.int32, device="cuda")
        if c["op"] == "attention_backward":
            out, s["lse"] = _attend(s)
            s["out"] = torch.empty((c["batch"], c["q_len"], c["heads"], c["dim"]), dtype=dt, device="cuda").transpose(1, 2).copy_(out)
            del out
            s["grad"] = _heads(g, c, c["heads"], c["q_len"])
            s["into"] = {"dq": torch.empty_like(s["q"]), "dk": torch.empty_like(s["k"]), "dv": torch.empty_like(s["v"])}
        else:
            s["into"] = {"out": torch.empty_like(s["q"]), "lse": torch.empty((c["batch"], c["heads"], c["q_len"]), device="cuda")}
    elif c["op"] == "rotary":
        s["q"], s["k"] = _heads(g, c, c["heads"], c["length"]), _heads(g, c, c["kv_heads"], c["length"])
        at = torch.randint(0, c["far"] + 1, (c["batch"], 1), generator=g, device="cuda") if c["far"] else torch.zeros((c["batch"], 1), dtype=torch.int64, device="cuda")
        s["positions"] = (at + torch.arange(c["length"], device="cuda")).to(torch.int32)
        s["into"] = {"q": torch.empty_like(s["q"]), "k": torch.empty_like(s["k"])}
    else:
        m, k, n = c["rows"], c["inner"], c["columns"]

        def normal(*shape, scale=1.0):
            return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt)

        s["a"] = normal(m, k)
        s["b"] = normal(n, k, scale=k ** -0.5).t() if c["transposed"] else normal(k, n, scale=k ** -0.5)
        if c["op"] == "product":
            s["bias"] = normal(n, scale=0.1)
            s["residual"] = normal(m, n) if c["residual"] else None
            s["into"] = {"out": torch.empty((m, n), dtype=dt, device="cuda")}
            if c["keep"]:
                s["into"]["pre"] = torch.empty((m, n), dtype=dt, device="cuda")
        else:
            s["pre"], s["grad"] = normal(m, n), normal(m, n)
            s["into"] = {"dz": torch.empty((m, n), dtype=dt, device="cuda"), "da": torch.empty((m, k), dtype=dt, device="cuda"),
                         "db": torch.empty((k, n), dtype=dt, device="cuda"), "dbias": torch.empty((n,), dtype=dt, device="cuda")}
    if own:
        s["call"] = _bind(s)    # the framework's tensors are descriptors; a program that holds the tensors holds these
        torch.cuda.synchronize()
    return s


def run(state):
    if own:
        entry, arguments, check = state["call"][:3]
        check(entry(*arguments))
        return state["into"]
    c = state["case"]
    dt = DTYPES[c["dtype"]]
    if c["op"] == "attention":
        out, lse = _attend(state)
        return {"out": out.to(dt), "lse": lse}
    if c["op"] == "attention_backward":
        dq, dk, dv = _attend_backward(state)
        return {"dq": dq.to(dt), "dk": dk.to(dt), "dv": dv.to(dt)}
    if c["op"] == "rotary":
        cos, sin = _turns(c, state["positions"])
        return {"q": _rotate(state["q"].float(), cos, sin, c).to(dt), "k": _rotate(state["k"].float(), cos, sin, c).to(dt)}
    if c["op"] == "product":
        z = state["a"].float() @ state["b"].float() + state["bias"].float()
        y = _activate(z, c["activation"])
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return {"out": y.to(dt), "pre": z.to(dt)} if c["keep"] else {"out": y.to(dt)}
    dz = state["grad"].float() * _slope(state["pre"].float(), c["activation"])
    return {"dz": dz.to(dt), "da": (dz @ state["b"].float().t()).to(dt), "db": (state["a"].float().t() @ dz).to(dt), "dbias": dz.sum(0).to(dt)}


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _visible(s):
    """[batch, 1, 1, q_len, k_len]: which key a query sees."""
    c = s["case"]
    lengths = torch.full((c["batch"],), c["k_len"], device="cuda") if s["lengths"] is None else s["lengths"].long()
    starts = lengths - c["q_len"] if s["starts"] is None else s["starts"].long()
    p = (starts[:, None] + torch.arange(c["q_len"], device="cuda"))[:, None, None, :, None]
    j = torch.arange(c["k_len"], device="cuda")
    seen = (j < lengths[:, None, None, None, None]) & (p >= 0)
    if c["causal"]:
        seen = seen & (j <= p)
    if c["window"]:
        seen = seen & (((p - j).abs() < c["window"]) | (j < c["sinks"]))
    return seen


def _grouped(x, kv_heads):
    return x.float().reshape(x.shape[0], kv_heads, -1, x.shape[2], x.shape[3])


def _attend(s):
    c = s["case"]
    q = _grouped(s["q"], c["kv_heads"])
    scores = torch.matmul(q.flatten(2, 3), s["k"].float().transpose(2, 3).contiguous()).unflatten(2, q.shape[2:4])
    scores = (scores * c["dim"] ** -0.5).masked_fill_(~_visible(s), float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    weights = (scores - top).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.flatten(2, 3), s["v"].float()).unflatten(2, q.shape[2:4])
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.flatten(1, 2), (top + total.log()).flatten(1, 2).squeeze(-1)


def _attend_backward(s):
    c = s["case"]
    q, grad = _grouped(s["q"], c["kv_heads"]), _grouped(s["grad"], c["kv_heads"])
    k, v = s["k"].float().contiguous(), s["v"].float().contiguous()
    scores = torch.matmul(q.flatten(2, 3), k.transpose(2, 3).contiguous()).unflatten(2, q.shape[2:4]) * c["dim"] ** -0.5
    lse = s["lse"].reshape(*q.shape[:4], 1)
    weights = torch.where(_visible(s), (scores - lse).exp_(), torch.zeros((), device="cuda"))
    delta = (grad * _grouped(s["out"], c["kv_heads"])).sum(-1, keepdim=True)
    dscores = weights * (torch.matmul(grad.flatten(2, 3), v.transpose(2, 3).contiguous()).unflatten(2, q.shape[2:4]) - delta) * c["dim"] ** -0.5
    dq = torch.matmul(dscores.flatten(2, 3), k).unflatten(2, q.shape[2:4]).flatten(1, 2)
    dk = torch.matmul(dscores.flatten(2, 3).transpose(2, 3).contiguous(), q.flatten(2, 3))
    dv = torch.matmul(weights.flatten(2, 3).transpose(2, 3).contiguous(), grad.flatten(2, 3))
    return dq, dk, dv


def _scaling(c):
    """(base, factor, original length, turns below which a frequency is divided, turns above which it is kept)"""
    return 10000.0, 8.0, 4096.0, 1.0, 32.0


def _turns(c, positions):
    """cos and sin of every angle, [batch, 1, length, rotated / 2]; the angles of far positions need 64 bits."""
    base, factor, original, low, high = _scaling(c)
    r = c["rotated"]
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    if c["scaling"] == "base":
        base = base * factor ** (r / (r - 2)) if r > 2 else base
    f = base ** (-2.0 * i / r)
    if c["scaling"] == "linear":
        f = f / factor
    if c["scaling"] == "parts":
        kept = ((original * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * (kept + (1 - kept) / factor)
    angle = positions.double()[:, None, :, None] * f
    return angle.cos().float(), angle.sin().float()


def _rotate(x, cos, sin, c):
    r = c["rotated"]
    if c["inverse"]:
        sin = -sin
    part = x[..., :r]
    a, b = (part[..., 0::2], part[..., 1::2]) if c["interleaved"] else part.chunk(2, -1)
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), -1).flatten(-2) if c["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., r:]), -1)


def _activate(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        e = 1 / (1 + torch.exp(-z))
        return e * (1 + z * (1 - e))
    return torch.ones_like(z)


# ---- the framework's calls ------------------------------------------------------------------------------------------

_context = None


def _bind(s):
    """The call of a case: its entry point, its arguments, what reads the status, and what the arguments point to."""
    from aix_amd import kernels as K
    global _context
    if _context is None:
        _context = K.Context(torch.cuda.current_device())
    names = {torch.float32: K.F32, torch.float16: K.F16, torch.bfloat16: K.BF16, torch.int32: K.I32}
    c, into = s["case"], s["into"]
    kept = []

    def tensor(t):
        if t is None:
            return None
        kept.append(K.tensor(t.data_ptr(), names[t.dtype], t.shape, t.stride()))
        return ctypes.byref(kept[-1])

    def pointer(t):
        if t is None:
            return None
        tensor(t)
        return ctypes.pointer(kept[-1])

    h, lib = _context.handle, _context.lib
    if c["op"] in ("attention", "attention_backward"):
        spec = K.AttentionSpec(scale=c["dim"] ** -0.5, causal=c["causal"], window=c["window"], sinks=c["sinks"],
                               lengths=pointer(s["lengths"]), starts=pointer(s["starts"]))
        kept.append(spec)
        q, k, v = tensor(s["q"]), tensor(s["k"]), tensor(s["v"])
        if c["op"] == "attention":
            return lib.aixk_attention, (h, q, k, v, ctypes.byref(spec), tensor(into["out"]), tensor(into["lse"])), K.check, kept
        return lib.aixk_attention_backward, (h, tensor(s["grad"]), q, k, v, tensor(s["out"]), tensor(s["lse"]), ctypes.byref(spec),
                                             tensor(into["dq"]), tensor(into["dk"]), tensor(into["dv"])), K.check, kept
    if c["op"] == "rotary":
        base, factor, original, low, high = _scaling(c)
        spec = K.RotarySpec(dims=c["rotated"], interleaved=c["interleaved"], inverse=c["inverse"], scaling=SCALINGS.index(c["scaling"]), base=base,
                            factor=factor, original_length=original, low_turns=low, high_turns=high, magnitude=1.0)
        kept.append(spec)
        return lib.aixk_rotary, (h, tensor(s["q"]), tensor(s["k"]), tensor(s["positions"]), ctypes.byref(spec), tensor(into["q"]), tensor(into["k"])), K.check, kept
    act = ACTIVATIONS.index(c["activation"])
    if c["op"] == "product":
        spec = K.Epilogue(bias=pointer(s["bias"]), residual=pointer(s["residual"]), pre=pointer(into.get("pre")), activation=act)
        kept.append(spec)
        return lib.aixk_matmul_epilogue, (h, tensor(s["a"]), tensor(s["b"]), ctypes.byref(spec), tensor(into["out"])), K.check, kept
    return lib.aixk_matmul_epilogue_backward, (h, tensor(s["grad"]), tensor(s["a"]), tensor(s["b"]), tensor(s["pre"]), act,
                                               tensor(into["dz"]), tensor(into["da"]), tensor(into["db"]), tensor(into["dbias"])), K.check, kept


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def _pairs(c, lengths, starts):
    """(visible pairs of a query and a key, keys that anybody sees) over all sequences, for one head."""
    pairs = keys = 0
    for length, start in zip(lengths, starts):
        p = torch.arange(max(start, 0), start + c["q_len"], dtype=torch.int64)
        if not len(p) or length <= 0:
            continue
        high = torch.minimum(p, torch.tensor(length - 1)) if c["causal"] else torch.full_like(p, length - 1)
        if not c["window"]:
            n = high + 1
            keys += int(high.max()) + 1
        else:
            low = (p - c["window"] + 1).clamp(min=0)
            if not c["causal"]:
                high = torch.minimum(high, p + c["window"] - 1)
            recent = (high - low + 1).clamp(min=0)
            first = torch.minimum(torch.full_like(p, min(c["sinks"], length)), (p + 1) if c["causal"] else torch.full_like(p, length))
            n = recent + torch.minimum(first, low)
            keys += int(min(max(0, int(high.max()) - int(low.min()) + 1) + min(int(first.max()), int(low.min())), length))
        pairs += int(n.sum())
    return pairs, keys


def work(case):
    c, size = case, SIZE[case["dtype"]]
    if c["op"] in ("attention", "attention_backward"):
        # the drawn lengths differ from seed to seed: half of the capacity on average, the start as the case has it
        lengths = [c["k_len"] // 2 if c["ragged"] else c["k_len"]] * c["batch"]
        starts = [0 if c["ragged"] and c["q_len"] == c["k_len"] else n - c["q_len"] for n in lengths]
        pairs, keys = _pairs(c, lengths, starts)
        rows, q = c["batch"] * c["heads"] * c["q_len"], c["batch"] * c["heads"] * c["q_len"] * c["dim"] * size
        cache = keys * c["kv_heads"] * c["dim"] * size
        if c["op"] == "attention":
            return {"bytes": 2 * q + 2 * cache + 4 * rows, "flops": 4.0 * pairs * c["heads"] * c["dim"]}
        return {"bytes": 4 * q + 4 * cache + 4 * rows, "flops": 10.0 * pairs * c["heads"] * c["dim"]}
    if c["op"] == "rotary":
        n = c["batch"] * (c["heads"] + c["kv_heads"]) * c["length"]
        return {"bytes": 2 * n * c["dim"] * size + 4 * c["batch"] * c["length"], "flops": 3.0 * n * c["rotated"]}
    m, k, n = c["rows"], c["inner"], c["columns"]
    if c["op"] == "product":
        return {"bytes": size * (m * k + k * n + n + m * n * (1 + c["residual"] + c["keep"])), "flops": 2.0 * m * n * k}
    return {"bytes": size * (2 * m * k + 2 * k * n + n + 3 * m * n), "flops": 4.0 * m * n * k}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["op"] in ("attention", "attention_backward"):
        return _exact_attention(c, s)
    if c["op"] == "rotary":
        return _exact_rotary(c, s)
    a, b = s["a"].double(), s["b"].double()
    if c["op"] == "product":
        z = torch.addmm(s["bias"].double(), a, b)
        y = {"none": lambda: z, "relu": lambda: torch.maximum(z, torch.zeros_like(z)), "silu": lambda: z * torch.sigmoid(z),
             "gelu": lambda: z * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3))}[c["activation"]]()
        if c["residual"]:
            y = y + s["residual"].double()
        return {"out": y, "pre": z} if c["keep"] else {"out": y}
    z = s["pre"].double().requires_grad_()
    y = {"relu": lambda: torch.relu(z), "silu": lambda: z * torch.sigmoid(z),
         "gelu": lambda: z * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3))}[c["activation"]]()
    dz, = torch.autograd.grad(y, z, s["grad"].double())
    return {"dz": dz, "da": dz @ b.T, "db": a.T @ dz, "dbias": dz.sum(0)}


def _exact_attention(c, s):
    group = c["heads"] // c["kv_heads"]
    back = c["op"] == "attention_backward"
    q64, k64, v64 = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k", "v"))
    out, lse = torch.zeros_like(q64), torch.full(q64.shape[:3], float("-inf"), dtype=torch.float64, device="cuda")
    for b in range(c["batch"]):
        length = c["k_len"] if s["lengths"] is None else int(s["lengths"][b])
        start = length - c["q_len"] if s["starts"] is None else int(s["starts"][b])
        p, j = torch.arange(start, start + c["q_len"], device="cuda")[:, None], torch.arange(length, device="cuda")[None, :]
        hidden = (p < 0) | torch.zeros_like(j, dtype=torch.bool)
        if c["causal"]:
            hidden = hidden | (j > p)
        if c["window"]:
            hidden = hidden | (((j <= p - c["window"]) | (j >= p + c["window"])) & (j >= c["sinks"]))
        rows = (~hidden).any(1) if length else torch.zeros(c["q_len"], dtype=torch.bool, device="cuda")
        if not bool(rows.any()):
            continue
        hidden = hidden[rows]
        for h in range(c["heads"]):
            q, k, v = s["q"][b, h].double()[rows], s["k"][b, h // group, :length].double(), s["v"][b, h // group, :length].double()
            x = (q @ k.T / c["dim"] ** 0.5).masked_fill(hidden, float("-inf"))
            if not back:
                lse[b, h, rows] = torch.logsumexp(x, 1)
                out[b, h, rows] = torch.softmax(x, 1) @ v
                continue
            w = torch.exp(x - s["lse"][b, h].double()[rows][:, None])
            grad = s["grad"][b, h].double()[rows]
            dx = w * (grad @ v.T - (grad * s["out"][b, h].double()[rows]).sum(1)[:, None]) / c["dim"] ** 0.5
            q64[b, h, rows] = dx @ k
            k64[b, h // group, :length] += dx.T @ q
            v64[b, h // group, :length] += w.T @ grad
    return {"dq": q64, "dk": k64, "dv": v64} if back else {"out": out, "lse": lse}


def _exact_rotary(c, s):
    base, factor, original, low, high = _scaling(c)
    r = c["rotated"]
    if c["scaling"] == "base" and r > 2:
        base *= factor ** (r / (r - 2))
    frequencies = []
    for i in range(r // 2):
        f = base ** (-2 * i / r)
        kept = min(1.0, max(0.0, (original * f / (2 * math.pi) - low) / (high - low)))
        frequencies.append(f / factor if c["scaling"] == "linear" else f * kept + f / factor * (1 - kept) if c["scaling"] == "parts" else f)
    angle = s["positions"].double()[:, None, :, None] * torch.tensor(frequencies, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones_like(angle), -angle if c["inverse"] else angle)
    result = {}
    for name in ("q", "k"):
        y = s[name].double()
        at = torch.arange(r // 2, device="cuda")
        first, second = (2 * at, 2 * at + 1) if c["interleaved"] else (at, at + r // 2)
        z = torch.complex(y[..., first], y[..., second]) * turn
        y = y.clone()
        y[..., first], y[..., second] = z.real, z.imag
        result[name] = y
    return result
