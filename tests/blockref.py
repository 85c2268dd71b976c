"""Plain 64-bit implementations of the transformer-block operators, and how far a result of the kernels may be from them.

Bounds count roundings: one to an element type is off by at most half a step, eps / 2 of the value (and half of the
smallest subnormal, which matters for f16 only); sums in f32 add 2^-24 of the sum of magnitudes per term."""
import math

import numpy as np

import aixtest as T
from oracle import cpuref as O

HALF = {O.F32: 2.0 ** -24, O.F16: 2.0 ** -11, O.BF16: 2.0 ** -8}
TINY = {O.F32: 2.0 ** -150, O.F16: 2.0 ** -25, O.BF16: 2.0 ** -134}
U32 = 2.0 ** -24
# The exponential's results below the smallest normal f32 become zeros, and so may f32 operands of the matrix unit: a weight
# or a score's gradient of any type may be off by 2^-126 on top of its relative error.
FLUSH = 2.0 ** -126


def visible(batch, queries, keys, causal, window, sinks, lengths, starts):
    """[batch, queries, keys] truth values."""
    lengths = np.full(batch, keys) if lengths is None else np.clip(np.asarray(lengths, np.int64), 0, keys)
    starts = lengths - queries if starts is None else np.asarray(starts, np.int64)
    p = (starts[:, None] + np.arange(queries))[:, :, None]
    j = np.arange(keys)[None, None, :]
    seen = (j < lengths[:, None, None]) & (p >= 0)
    if causal:
        seen &= j <= p
    if window:
        seen &= (np.abs(p - j) < window) | (j < sinks)
    return seen


def attention(q, k, v, seen, scale, dtype):
    """q [b, h, s, d], k and v [b, hk, t, d] in float64 -> out, lse and their bounds."""
    b, h, s, d = q.shape
    group = h // k.shape[1]
    out, lse = np.zeros_like(q), np.full((b, h, s), -np.inf)
    out_far, lse_far = np.zeros_like(q), np.zeros((b, h, s))
    for i in range(b):
        for j in range(h):
            kk, vv, ok = k[i, j // group], v[i, j // group], seen[i]
            rows = ok.any(1)
            if not rows.any():
                continue
            kk, vv = np.where(ok.any(0)[:, None], kk, 0), np.where(ok.any(0)[:, None], vv, 0)
            x = np.where(ok, scale * (q[i, j] @ kk.T), -np.inf)
            top = np.where(rows, x.max(1, initial=-np.inf), 0)
            w = np.exp(x - top[:, None])
            total = w.sum(1)
            w = np.divide(w, total[:, None], out=np.zeros_like(w), where=total[:, None] > 0)
            out[i, j] = w @ vv
            lse[i, j] = np.where(rows, top + np.log(np.where(rows, total, 1)), -np.inf)
            e = score_far(q[i, j], kk, scale, ok, d)
            n = ok.sum(1)
            p_half = HALF[dtype] if dtype != O.F32 else 0.0
            part = (p_half + 2 * e + (n + 16) * U32)[:, None] * (w @ np.abs(vv)) + (FLUSH + (TINY[dtype] if dtype == O.F16 else 0)) * np.abs(vv).sum(0)
            out_far[i, j] = part + HALF[dtype] * np.abs(out[i, j]) + TINY[dtype]
            lse_far[i, j] = e + (n + 16) * U32 + 4 * U32 * np.abs(np.where(rows, lse[i, j], 0))
    return out, lse, out_far, lse_far


def score_far(q, k, scale, ok, d):
    """[queries]: how far an exponent may be: f32 sums of d products, the scaling, and the argument of the exponential."""
    mass = scale * (np.abs(q) @ np.abs(k).T)
    size = np.abs(scale * (q @ k.T))
    return np.where(ok, (d + 4) * U32 * mass + 6 * U32 * size, 0).max(1, initial=0) + 4 * U32


def attention_backward(grad, q, k, v, out, lse, seen, scale, dtype):
    """-> dq, dk, dv and their bounds."""
    b, h, s, d = q.shape
    group = h // k.shape[1]
    got = [np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)]
    far = [np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)]
    p_half, tiny = HALF[dtype] if dtype != O.F32 else 0.0, FLUSH + (TINY[dtype] if dtype == O.F16 else 0.0)
    for i in range(b):
        for j in range(h):
            c, ok = j // group, seen[i]
            keys = ok.any(0)[:, None]
            kk, vv, qq, gg, yy = np.where(keys, k[i, c], 0), np.where(keys, v[i, c], 0), q[i, j], grad[i, j], out[i, j]
            x = scale * (qq @ kk.T)
            stat = np.where(np.isfinite(lse[i, j]), lse[i, j], np.inf)[:, None]
            w = np.where(ok, np.exp(np.minimum(x - stat, 700)), 0)
            dp, delta = gg @ vv.T, (gg * yy).sum(1)[:, None]
            ds = w * (dp - delta)
            got[0][i, j] = scale * (ds @ kk)
            got[1][i, c] += scale * (ds.T @ qq)
            got[2][i, c] += w.T @ gg
            e = score_far(qq, kk, scale, ok, d)[:, None] + 4 * U32 * np.abs(np.where(np.isfinite(stat), stat, 0))
            dp_far = (d + 4) * U32 * (np.abs(gg) @ np.abs(vv).T + (np.abs(gg) * np.abs(yy)).sum(1)[:, None])
            w_far = (p_half + e) * w + tiny * ok
            ds_far = (p_half + e + 4 * U32) * np.abs(ds) + w * dp_far + (tiny + FLUSH * np.abs(dp - delta)) * ok
            nk, nq = ok.sum(1)[:, None], (ok.sum(0) * group)[:, None]
            far[0][i, j] = scale * (ds_far @ np.abs(kk) + (nk + 8) * U32 * (np.abs(ds) @ np.abs(kk)))
            far[1][i, c] += scale * (ds_far.T @ np.abs(qq) + (nq + 8) * U32 * (np.abs(ds).T @ np.abs(qq)))
            far[2][i, c] += w_far.T @ np.abs(gg) + (nq + 8) * U32 * (w.T @ np.abs(gg))
    return got, [f + HALF[dtype] * np.abs(g) + TINY[dtype] for f, g in zip(far, got)]


def check(got, want, far, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, f"{what}: {got.shape} against {want.shape}"
    with np.errstate(invalid="ignore"):
        same = (got == want) | (np.abs(got - want) <= far)
    if not same.all():
        at = tuple(int(x) for x in np.argwhere(~same)[0])
        raise AssertionError(f"{what}: {int((~same).sum())} of {got.size} beyond their bounds; first at {at}: got {got[at]!r}, want {want[at]!r} +- {far[at]!r}")


# ---- device tensors -------------------------------------------------------------------------------------------------

class Box:
    """A host array of an element type behind a descriptor: a view (permutation, padding) of a dense block on the device."""

    def __init__(self, gpu, K, dtype, shape, values=None, order=None, pad=0, offset=0, fill=None):
        """order: the memory order of the dims; pad: elements added to the innermost memory dim; offset: elements before the view."""
        self.gpu, self.dtype, self.shape = gpu, dtype, tuple(shape)
        order = list(range(len(shape))) if order is None else list(order)
        extent = [shape[d] for d in order]
        if pad and extent:
            extent[-1] += pad
        strides, run = [0] * len(shape), 1
        for n in reversed(range(len(order))):
            strides[order[n]], run = run, run * extent[n]
        self.offset, self.count = offset, run + offset
        self.strides = strides
        store = T_zeros(dtype, self.count) if fill is None else T_round(np.full(self.count, fill), dtype)
        self.store = store
        self.before = None
        if values is not None:
            self.view(store)[...] = T_round(np.asarray(values, np.float64), dtype)
        self.ptr = gpu.raw(max(store.nbytes, 1))
        gpu.ctx.upload(self.ptr, store)
        self.before = store.copy()
        self.desc = K.tensor(self.ptr, dtype, shape, strides, offset)

    def view(self, store):
        return np.lib.stride_tricks.as_strided(store[self.offset:] if store.size > self.offset else store[:0], self.shape,
                                               [x * store.itemsize for x in self.strides])

    def fetch(self):
        """The view's values in float64; what lies between must be as it was."""
        raw = np.empty_like(self.store)
        if raw.nbytes:
            self.gpu.ctx.download(raw, self.ptr)
        used = np.zeros(self.store.size, bool)
        np.lib.stride_tricks.as_strided(used[self.offset:], self.shape, self.strides)[...] = True
        assert np.array_equal(raw[~used], self.before[~used]), "elements outside of the view were written"
        return T_float(self.view(raw), self.dtype)

    def values(self):
        return T_float(self.view(self.before), self.dtype)


def T_zeros(dtype, n):
    return np.zeros(n, {O.F32: np.float32, O.F16: np.float16, O.BF16: np.uint16, O.I32: np.int32}[dtype])


def T_round(x, dtype):
    if dtype == O.BF16:
        from aix_amd.workloads import round_to_bf16_bits
        return round_to_bf16_bits(np.asarray(x, np.float32))
    return np.asarray(x).astype({O.F32: np.float32, O.F16: np.float16, O.I32: np.int32}[dtype])


def T_float(x, dtype):
    if dtype == O.BF16:
        return (np.ascontiguousarray(x).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return np.array(x, np.float64)


# ---- rotary positions -----------------------------------------------------------------------------------------------

def rotary(x, positions, dims, interleaved, inverse, frequencies, magnitude, dtype):
    """x [b, h, s, d]; positions [b, s] -> the turned tensor and its bound: f32 sines and cosines, two products, one rounding."""
    angle = positions.astype(np.float64)[:, None, :, None] * np.asarray(frequencies)
    c, s = np.cos(angle) * magnitude, np.sin(angle) * magnitude * (-1 if inverse else 1)
    i = np.arange(dims // 2)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + dims // 2)
    out, far = x.copy(), np.zeros_like(x)
    out[..., first] = x[..., first] * c - x[..., second] * s
    out[..., second] = x[..., first] * s + x[..., second] * c
    # the fraction of a turn rounds to f32 (half a unit of at most half a turn: pi 2^-24), the functions are good to 2 units
    mass = (np.abs(x[..., first]) + np.abs(x[..., second])) * magnitude * 10 * U32 + np.abs(angle) * 2.0 ** -50
    far[..., first] = mass + HALF[dtype] * np.abs(out[..., first]) + TINY[dtype]
    far[..., second] = mass + HALF[dtype] * np.abs(out[..., second]) + TINY[dtype]
    return out, far


def frequencies(dims, scaling="plain", base=10000.0, factor=1.0, original=1.0, low=0.0, high=1.0):
    if scaling == "base" and dims > 2:
        base = base * factor ** (dims / (dims - 2))
    f = base ** (-2.0 * np.arange(dims // 2) / dims)
    if scaling == "linear":
        f = f / factor
    if scaling == "parts":
        kept = np.clip((original * f / (2 * math.pi) - low) / (high - low), 0, 1)
        f = f * (kept + (1 - kept) / factor)
    return f


# ---- products with an epilogue --------------------------------------------------------------------------------------

C_GELU = math.sqrt(2 / math.pi)


def _argument(z, act):
    return 2 * C_GELU * (z + 0.044715 * z ** 3) if act == "gelu" else z


def activate(z, act):
    """act(z), the size of its slope at most, and its own rounding: the exponent is good to a few units of itself."""
    if act == "relu":
        return np.maximum(z, 0), 1.0, 0 * z
    if act == "none":
        return z, 1.0, 0 * z
    w = _argument(z, act)
    y = z / (1 + np.exp(-np.clip(w, -700, 700)))
    return y, 1.2, np.abs(y) * (np.minimum(np.abs(w), 80) + 8) * 6 * U32 + 1e-30


def slope(z, act):
    if act == "relu":
        return (z > 0).astype(np.float64), 0 * z
    if act == "none":
        return np.ones_like(z), 0 * z
    w = _argument(z, act)
    e = np.exp(-np.clip(w, -700, 700))            # (the clip keeps e s at 1 on the far side and 0 on the near one)
    s = 1 / (1 + e)
    inner = 2 * C_GELU * (1 + 3 * 0.044715 * z ** 2) if act == "gelu" else 1.0
    bend = z * s * (e * s) * inner
    return s + bend, (np.minimum(np.abs(w), 80) + 8) * 6 * U32 * (s + np.abs(bend)) + 4 * U32


def product_far(x, y, k):
    """an f32 sum of k products; f32 operands go through the matrix unit as three bf16 planes, off by 2^-22 of a product"""
    return ((k + 8) * U32 + 2.0 ** -22) * (np.abs(x) @ np.abs(y))


def matmul_epilogue(a, b, bias, residual, act, dtype):
    z = a @ b + (bias if bias is not None else 0)
    z_far = product_far(a, b, a.shape[1]) + 2 * U32 * (np.abs(z) + np.abs(bias if bias is not None else 0))
    y, steep, y_far = activate(z, act)
    out = y + (residual if residual is not None else 0)
    far = steep * z_far + y_far + 2 * U32 * (np.abs(y) + np.abs(out))
    return out, far + HALF[dtype] * np.abs(out) + TINY[dtype], z, z_far + HALF[dtype] * np.abs(z) + TINY[dtype]


def matmul_epilogue_backward(grad, a, b, pre, act, dtype):
    s, s_far = slope(pre, act) if pre is not None else (np.ones_like(grad), 0 * grad)
    dz = grad * s
    exact_far = np.abs(grad) * s_far + U32 * np.abs(dz)
    dz_far = exact_far + HALF[dtype] * np.abs(dz) + TINY[dtype]
    m, n = grad.shape
    da, db, dbias = dz @ b.T, a.T @ dz, dz.sum(0)
    h, t = HALF[dtype], TINY[dtype]
    return (dz, da, db, dbias), (dz_far, dz_far @ np.abs(b).T + product_far(dz, b.T, n) + h * np.abs(da) + t,
                                 np.abs(a).T @ dz_far + product_far(a.T, dz, m) + h * np.abs(db) + t,
                                 exact_far.sum(0) + (m + 8) * U32 * np.abs(dz).sum(0) + h * np.abs(dbias) + t)
