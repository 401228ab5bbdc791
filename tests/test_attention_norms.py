"""window_attention's outputs and gradients by their norms: each whole, and for each 128 tokens of each head (a tile of a workgroup),
so that a part of the rows or keys that is left out shows.

Tolerances: a rounding to bfloat16 is off by a uniform part of at most half a step of 2^-7 of the value's binade, by 2^-7 / sqrt(12)
of it in the mean square. Three of them at most meet in an output, independent of one another: the probabilities' or the scores'
gradients', the probabilities' in delta, and the output's own: sqrt(3) 2^-7 / sqrt(12) = 2^-8 of a norm. In float32 the largest
error is a probability's, its exponent's: some 16 of base 2, of sums of up to 128 terms, below 128 roundings of 2^-24."""
import ctypes as C

import pytest
import torch

import psgd_pro_amd as P
from psgd_pro_amd import _lib as L
from test_attention import DTYPES, inputs, reference

pytestmark = pytest.mark.gpu
NORM = {torch.float32: 2.0 ** -17, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(autouse=True)
def _lib(hip):
    return hip


def by_norm(out, ref, bound, what):
    off, size = (out.double() - ref).square(), ref.square()
    assert float(off.sum().sqrt()) <= bound * float(size.sum().sqrt()), (what, float((off.sum() / size.sum()).sqrt()))
    for t in range(0, out.shape[1], 128):
        e, s = (x[:, t:t + 128].sum((1, 3)).sqrt() for x in (off, size))
        assert bool((e <= bound * s).all()), (what, t, float((e / s).max()))


def run(q, k, v, do, **kw):
    refs, _ = reference(q, k, v, do, **kw)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = P.window_attention(*leaves, **kw)
    for name, out, ref in zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do)), refs):
        by_norm(out, ref, NORM[q.dtype], name)


def parts(b, n, h, kv, d, dtype, window, sinks):
    """Whether tiles of the dk, dv pass are cut: its workspace holds more than the rows' two numbers then."""
    a = L.WindowAttention(batch=b, n=n, m=n, heads=h, kv_heads=kv, d=d, dtype=L.dtype_code(dtype), window=window or 0, sinks=sinks, scale=0.1)
    size = C.c_size_t(0)
    g = L.WindowAttentionGrads(L.Heads(1 << 16, 0, 0, 0), 1 << 16, 1 << 16, 1 << 16)
    L.check(L.lib().psgdk_window_attention_backward(C.byref(a), C.byref(g), None, C.byref(size), None))
    return size.value > 2 * (4 * b * n * h + 256)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,n,h,kv,d,window,sinks,cut", [
    (2, 300, 3, 1, 128, None, 0, True), (1, 2900, 4, 1, 128, 100, 5, True), (1, 1600, 8, 4, 128, None, 0, True), (8, 1024, 8, 8, 128, None, 0, False),
    (1, 3001, 2, 2, 64, 300, 130, True), (8, 1024, 8, 8, 64, 200, 0, False), (1, 1500, 4, 2, 96, 200, 3, True), (8, 1024, 8, 8, 96, None, 0, False),
    (1, 2700, 2, 2, 32, 90, 4, True), (8, 1024, 8, 8, 32, None, 0, False)])
def test_norms_of_outputs_and_gradients(dtype, b, n, h, kv, d, window, sinks, cut):
    assert parts(b, n, h, kv, d, dtype, window, sinks) == cut
    run(*inputs(b, n, n, h, kv, d, dtype), window=window, sinks=sinks)


@pytest.mark.parametrize("n,h,kv,d,window,sinks", [(1000, 2, 2, 64, None, 0), (1000, 4, 2, 128, 100, 5), (700, 2, 1, 32, 90, 4), (700, 2, 2, 96, 200, 3)])
def test_gradients_where_values_have_a_mean(n, h, kv, d, window, sinks):
    """Values around 16: o is as large, and delta, the sum of o and its gradient, has to be right far below o's own rounding (left to
    it, gradients of queries and keys are .03 to .04 off)."""
    q, k, v, do = inputs(1, n, n, h, kv, d, torch.bfloat16)
    run(q, k, v + 16, do, window=window, sinks=sinks)
