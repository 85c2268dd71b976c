"""The memory that the backward pass of attention takes for partial sums of many leading keys on many heads."""
import ctypes as C

import numpy as np
import pytest

import blockref as R
import gpuharness as G
from aix_amd import kernels as K
from oracle import cpuref as O

from test_gpu_attention import Case

pytestmark = pytest.mark.gpu


def test_many_leading_keys_on_many_heads():
    """Per query tile a copy of the leading keys' gradients would be 2.8 GB here; the gradients themselves are 0.27 GB in f32."""
    import torch
    gpu = G.Gpu()                                              # a context without workspaces
    batch, heads, length, d = 4, 16, 8192, 64
    shape = (batch, heads, length, d)
    count = int(np.prod(shape))
    data = [gpu.raw(2 * count) for _ in range(8)]
    rng = np.random.default_rng(3)
    bits = R.T_round(rng.standard_normal(count // batch), O.BF16)
    for p in data[:4]:
        for b in range(batch):
            gpu.ctx.upload(p + 2 * b * bits.size, np.roll(bits, 17 * b + data.index(p)))
    q, k, v, grad, out, dq, dk, dv = [K.tensor(p, O.BF16, shape) for p in data]
    lse = K.tensor(gpu.raw(4 * batch * heads * length), O.F32, shape[:3])
    spec = K.AttentionSpec(scale=0.125, causal=1, window=256, sinks=4096, lengths=None, starts=None)
    G.run_gpu(gpu, "aixk_attention", G.ref(q), G.ref(k), G.ref(v), C.byref(spec), G.ref(out), G.ref(lse))
    gpu.ctx.sync()
    before = torch.cuda.mem_get_info()[0]
    G.run_gpu(gpu, "aixk_attention_backward", G.ref(grad), G.ref(q), G.ref(k), G.ref(v), G.ref(out), G.ref(lse), C.byref(spec), G.ref(dq), G.ref(dk), G.ref(dv))
    gpu.ctx.sync()
    assert before - torch.cuda.mem_get_info()[0] <= 600 << 20
    # the sum of dv over the keys is the sum of the gradients over the queries (the weights of a query add up to one): every
    # weight rounded to bf16 (2^-8), every dv rounded to bf16, over 8192 of each
    total = np.empty(count // batch // heads, np.uint16)
    gpu.ctx.download(total, data[7])
    got = R.T_float(total, O.BF16).reshape(length, d)
    sent = np.empty_like(total)
    gpu.ctx.download(sent, data[3])
    want = R.T_float(sent, O.BF16).reshape(length, d)
    far = 2.0 ** -8 * np.abs(want).sum(0) + 2.0 ** -8 * np.abs(got).sum(0)
    R.check(got.sum(0), want.sum(0), far, "sums of dv")
    gpu.release()
    gpu.close()


@pytest.mark.parametrize("heads,kv,sq,sinks,window,d", [(48, 48, 900, 300, 100, 64), (40, 20, 1200, 200, 64, 128), (2, 2, 1500, 400, 50, 64), (3, 3, 1100, 130, 40, 256)])
def test_leading_keys_with_shares_and_without(heads, kv, sq, sinks, window, d):
    gpu = G.Gpu()
    for causal in (True, False):
        case = Case(gpu, O.BF16, 1, heads, kv, sq, sq, d, causal=causal, window=window, sinks=sinks)
        case.forward()
        case.backward()
        case.check_backward(f"{heads} heads, {sinks} leading keys, causal {causal}")
        case.release()
    gpu.close()
