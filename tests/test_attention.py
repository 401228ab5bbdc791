"""window_attention on the GPU against a plain implementation in float64.

Tolerances are bounds of the rounding errors, computed next to the reference from the same magnitudes: U is the rounding of a
value to its storage type (half a unit of the last place), E fp32's; a sum of n terms in any order is within n E of the sum of
its terms' magnitudes. With bfloat16 the probabilities, their sum and the scores' gradients carry one U each besides."""
import math

import pytest
import torch

import psgd_pro_amd as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(autouse=True)
def _lib(hip):
    return hip


def rnd(shape, seed, dtype=torch.float32, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def within(out, ref, bound, what=""):
    assert out.shape == ref.shape, (what, out.shape, ref.shape)
    err = (out.double() - ref).abs()
    bad = ~(err <= bound + 1e-300)
    assert not bool(bad.any()), (what, int(bad.sum()), float((err / (bound + 1e-300)).nan_to_num(nan=9e9).max()))


def visible(b, n, m, window, sinks, lengths, starts):
    i, j = torch.arange(n, device=DEV), torch.arange(m, device=DEV)
    length = torch.full((b,), m, device=DEV) if lengths is None else lengths.clamp(0, m)
    start = torch.full((b,), m - n, device=DEV) if starts is None else starts
    pos = (start[:, None] + i)[:, None, :, None]
    see = (pos >= 0) & (pos < length[:, None, None, None]) & (j <= pos)
    return see if window is None else see & ((pos - j < window) | (j < sinks))


def reference(q, k, v, do, window=None, sinks=0, lengths=None, starts=None, scale=None):
    """((o, dq, dk, dv), their bounds), in float64; do None: o alone."""
    u = U[q.dtype] if q.dtype == torch.bfloat16 else 0.0
    store = U[q.dtype]
    b, n, h, d = q.shape
    m, kv = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    see = visible(b, n, m, window, sinks, lengths, starts)
    live = see.any(-1, keepdim=True)
    heads = lambda t: t.detach().double().permute(0, 2, 1, 3)  # noqa: E731  (batch, heads, tokens, d)
    many = lambda t: heads(t).repeat_interleave(h // kv, 1)  # noqa: E731
    # (what is not visible to anyone may hold anything)
    Q, K, V = (torch.where(ok, t, 0.0) for t, ok in ((heads(q), live), (many(k), see.any(2)[..., None]), (many(v), see.any(2)[..., None])))
    s = Q @ K.transpose(2, 3).contiguous() * scale
    size = Q.abs() @ K.abs().transpose(2, 3).contiguous() * scale
    s = torch.where(see, s, -math.inf)
    top = torch.where(live, s.amax(-1, keepdim=True), 0.0)
    p = torch.where(see, torch.exp(s - top), 0.0)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    # a probability's relative error: its score's (d products, scaled), the rounding of the exponent (its size in base 2, up to
    # the largest score's), the exponential's and the sum's
    far = torch.where(see, (s - top).abs() + size, 0.0).amax(-1, keepdim=True)
    eps = 2 * (d + 4) * E * torch.where(see, size, 0.0).amax(-1, keepdim=True) + (4 * far + 24 + 2 * m) * E
    o = p @ V
    A = p @ V.abs()
    back = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
    few = lambda t: t.unflatten(1, (kv, h // kv)).sum(2)  # noqa: E731
    err_o = (2 * u + 2 * eps + m * E) * A + store * o.abs()
    if do is None:
        return (back(o),), (back(err_o),)
    G = torch.where(live, heads(do), 0.0)
    dv = p.transpose(2, 3).contiguous() @ G
    dv_err = (p * (2 * u + 2 * eps + n * h * E)).transpose(2, 3).contiguous() @ G.abs()
    dp = G @ V.transpose(2, 3).contiguous()
    delta = (G * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    ds_err = ds.abs() * (2 * u + 2 * eps + 8 * E) + p * (2 * d * E * (G.abs() @ V.abs().transpose(2, 3).contiguous())
                                                         + (G.abs() * (err_o + 2 * d * E * o.abs())).sum(-1, keepdim=True))
    total = ds_err + ds.abs() * (m + n * h) * E
    dq, dq_err = ds @ K * scale, total @ K.abs() * scale
    dk, dk_err = few(ds.transpose(2, 3).contiguous() @ Q) * scale, few(total.transpose(2, 3).contiguous() @ Q.abs()) * scale
    outs = (o, dq, few(dv), dk)
    o, dq, dv, dk = (back(t) for t in (o, dq, few(dv), dk))
    errs = back(err_o), back(dq_err) + store * dq.abs(), back(dk_err) + store * dk.abs(), back(few(dv_err)) + store * dv.abs()
    return (o, dq, dk, dv), errs


def check(q, k, v, do, **kw):
    refs, bounds = reference(q, k, v, do, **kw)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = P.window_attention(*leaves, **kw)
    with torch.no_grad():
        assert torch.equal(o, P.window_attention(*leaves, **kw))
    outs = (o,) if do is None else (o, *torch.autograd.grad(o, leaves, do))
    for name, t, r, e in zip(("o", "dq", "dk", "dv"), outs, refs, bounds):
        assert t.dtype == q.dtype
        within(t, r, e, name)


def inputs(b, n, m, h, kv, d, dtype, seed=0, std=1.0):
    return (rnd((b, n, h, d), seed + 1, dtype, std), rnd((b, m, kv, d), seed + 2, dtype, std), rnd((b, m, kv, d), seed + 3, dtype),
            rnd((b, n, h, d), seed + 4, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,n,h,kv,d,window,sinks", [
    (1, 1, 1, 1, 8, None, 0), (2, 2, 2, 1, 16, 1, 0), (1, 31, 3, 3, 24, None, 0), (1, 33, 4, 2, 40, 7, 1), (2, 64, 2, 2, 64, None, 0),
    (1, 65, 6, 2, 72, 64, 3), (3, 127, 2, 1, 80, None, 0), (1, 128, 4, 4, 96, 33, 40), (1, 129, 5, 1, 104, 500, 2),
    (1, 257, 8, 2, 128, 128, 129), (2, 300, 3, 1, 128, None, 0), (1, 2900, 4, 1, 128, 100, 5), (1, 3001, 2, 2, 64, 300, 130), (1, 700, 2, 2, 32, 90, 4), (1, 513, 12, 4, 56, 256, 0)])
def test_training_matches_float64(dtype, b, n, h, kv, d, window, sinks):
    q, k, v, do = inputs(b, n, n, h, kv, d, dtype)
    check(q, k, v, do, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 0), (20, 5), (1, 1), (1000, 1000)])
def test_padded_batch_whatever_the_padding_holds(dtype, window, sinks):
    """Lengths from none to all, and one out of range; behind them NaN and infinities in the inputs and the gradient."""
    b, n, h, kv, d = 6, 150, 4, 2, 64
    lengths = torch.tensor([0, 1, 64, 149, 150, 10 ** 12], device=DEV)
    q, k, v, do = inputs(b, n, n, h, kv, d, dtype)
    for i, (t, bad) in enumerate(((q, math.nan), (k, math.inf), (v, math.nan), (do, -math.inf))):
        for s in range(b):
            t[s, min(int(lengths[s]), n):] = bad
    check(q, k, v, do, window=window, sinks=sinks, lengths=lengths)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = P.window_attention(*leaves, window=window, sinks=sinks, lengths=lengths)
    for t in (o, *torch.autograd.grad(o, leaves, do)):
        for s in range(b):
            assert not t[s, min(int(lengths[s]), n):].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,n,m,h,kv,d,window,sinks", [
    (4, 1, 700, 8, 2, 128, None, 0), (3, 1, 1500, 2, 2, 64, 300, 4), (2, 7, 2000, 4, 1, 80, 1000, 4), (1, 1, 20000, 8, 1, 128, None, 0),
    (1, 16, 5000, 8, 2, 64, None, 0), (2, 40, 900, 4, 2, 96, 100, 2), (1, 65, 3000, 1, 1, 32, None, 0), (70, 1, 300, 3, 1, 40, 64, 1)])
def test_caches_and_short_queries(dtype, b, n, m, h, kv, d, window, sinks):
    """The last tokens of sequences of different lengths over caches with room behind them, which holds NaN."""
    q, k, v, do = inputs(b, n, m, h, kv, d, dtype)
    g = torch.Generator(device=DEV).manual_seed(9)
    lengths = torch.randint(max(n, m // 3), m + 1, (b,), generator=g, device=DEV)
    for s in range(b):
        k[s, lengths[s]:] = v[s, lengths[s]:] = math.nan
    check(q, k, v, do, window=window, sinks=sinks, lengths=lengths, starts=lengths - n)


def test_positions_outside_the_sequence_see_nothing():
    """Starts before the first token, behind the last, far outside 32 bits; more queries than keys."""
    q, k, v, do = inputs(6, 40, 100, 2, 1, 64, torch.float32)
    starts = torch.tensor([-20, 80, 100, -(10 ** 15), 10 ** 15, 60], device=DEV)
    check(q, k, v, do, starts=starts)
    q, k, v, do = inputs(2, 50, 20, 2, 1, 16, torch.bfloat16)
    check(q, k, v, do)
    check(q, k, v, do, window=3, sinks=2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_all_sizes(dtype):
    """Peaked rows (scores up to some 60 either side), with the largest far behind the first tiles; a scale of its own."""
    q, k, v, do = inputs(1, 400, 400, 2, 1, 64, dtype, std=2.5)
    check(q, k, v, do, window=250, sinks=10)
    check(q, k, v, do, scale=0.031)
    ramp = torch.arange(400, device=DEV).view(1, 400, 1, 1) / 40
    check((q * 0 + 1).to(dtype), (k * 0.01 + ramp).to(dtype), v, do)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    """Parts of one projection, heads first, slices on odd boundaries (copied), broadcast keys; an expanded gradient."""
    x = rnd((2, 90, 8, 64), 1, dtype)
    do = rnd((2, 90, 4, 64), 2, dtype)
    check(*x.split((4, 2, 2), 2), do)
    y = rnd((2, 8, 90, 64), 3, dtype).transpose(1, 2)
    check(y[:, :, :4], y[:, :, 4:6], y[:, :, 6:], do)
    z = rnd((2, 90, 8, 67), 4, dtype)[..., 1:65]
    check(*z.split((4, 2, 2), 2), do)
    one = rnd((2, 90, 1, 64), 5, dtype).expand(2, 90, 2, 64)
    check(x[:, :, :4], one, one.flip(1), rnd((1, 1, 1, 64), 6, dtype).expand(2, 90, 4, 64))
    check(x[:, :, :4], x[:, :, 4:6], x[:, :, 6:], rnd((2, 90, 4, 1), 7, dtype).expand(2, 90, 4, 64))


def test_a_long_cache_of_each_heads_tokens_is_read_in_place():
    b, m, h, kv, d = 1, 40000, 4, 2, 64  # heads 2.56 M elements apart
    q, do = rnd((b, 2, h, d), 70, torch.bfloat16), rnd((b, 2, h, d), 71, torch.bfloat16)
    kc, vc = (rnd((b, kv, m, d), s, torch.bfloat16).transpose(1, 2) for s in (72, 73))
    lengths = torch.tensor([m - 5], device=DEV)
    starts = lengths - 2
    ref, bounds = reference(q, kc, vc, None, 1000, 3, lengths, starts)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    o = P.window_attention(q, kc, vc, window=1000, sinks=3, lengths=lengths, starts=starts)
    assert torch.cuda.max_memory_allocated() - before < kc.numel() * 2  # (no copy of either cache)
    within(o, ref[0], bounds[0])
    leaves = [t.detach().requires_grad_() for t in (q, kc, vc)]
    grads = torch.autograd.grad(P.window_attention(*leaves, window=1000, sinks=3, lengths=lengths, starts=starts), leaves, do)
    near = [t.detach().contiguous().requires_grad_() for t in (q, kc, vc)]
    for x, y in zip(grads, torch.autograd.grad(P.window_attention(*near, window=1000, sinks=3, lengths=lengths, starts=starts), near, do)):
        assert torch.equal(x, y)


def test_offsets_beyond_32_bits():
    """A cache of 2^33 bytes: the window at its end, and the first tokens."""
    m, kv, d = 1 << 22, 8, 128
    k = torch.zeros(1, m, kv, d, device=DEV, dtype=torch.bfloat16)
    v = torch.zeros(1, m, kv, d, device=DEV, dtype=torch.bfloat16)
    k[:, -300:], v[:, -300:] = rnd((1, 300, kv, d), 1, k.dtype), rnd((1, 300, kv, d), 2, k.dtype)
    k[:, :5], v[:, :5] = rnd((1, 5, kv, d), 3, k.dtype), rnd((1, 5, kv, d), 4, k.dtype)
    q = rnd((1, 3, 16, d), 5, k.dtype)
    out = P.window_attention(q, k, v, window=200, sinks=5)
    near = torch.cat((k[:, :5], k[:, -300:]), 1), torch.cat((v[:, :5], v[:, -300:]), 1)
    refs, bounds = reference(q, *near, None, window=200, sinks=5)
    within(out, refs[0], bounds[0])


def test_empty_sizes():
    q, k, v, _ = inputs(2, 5, 7, 4, 2, 32, torch.float32)
    assert P.window_attention(q[:0], k[:0], v[:0]).shape == (0, 5, 4, 32)
    assert P.window_attention(q[:, :0], k, v).shape == (2, 0, 4, 32)
    leaves = [t.requires_grad_() for t in (q, k[:, :0].clone(), v[:, :0].clone())]
    o = P.window_attention(*leaves)
    assert not o.any()
    for g, t in zip(torch.autograd.grad(o.sum(), leaves), leaves):
        assert g.shape == t.shape and not g.any()


def test_gradients_against_differences():
    """Central differences of the float32 forward pass along random directions: their error is the third derivative's h^2 and
    the rounding of o over h."""
    q, k, v, do = inputs(2, 60, 60, 4, 2, 24, torch.float32)
    kw = dict(window=25, sinks=3, lengths=torch.tensor([60, 41], device=DEV))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(P.window_attention(*leaves, **kw), leaves, do)
    h = 2.0 ** -7
    for i in range(3):
        step = rnd(leaves[i].shape, 50 + i)
        ends = []
        for sign in (1, -1):
            args = [t.detach() + (sign * h * step if j == i else 0) for j, t in enumerate(leaves)]
            ends.append((P.window_attention(*args, **kw).double() * do).sum())
        want, got = (ends[0] - ends[1]) / (2 * h), (grads[i].double() * step).sum()
        size = (grads[i].double() * step).norm()
        assert abs(float(want - got)) < 40 * h * h * float(size) + 1e-6 * float(do.norm()) * math.sqrt(do.numel()) / h


def test_single_gradients_and_second_backward():
    q, k, v, do = inputs(1, 200, 200, 4, 2, 64, torch.bfloat16)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = P.window_attention(*leaves, window=50, sinks=1)
    all_three = torch.autograd.grad(o, leaves, do, retain_graph=True)
    for a, b in zip(all_three, torch.autograd.grad(o, leaves, do, retain_graph=True)):
        assert torch.equal(a, b)
    for i in range(3):
        only = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(P.window_attention(*only, window=50, sinks=1), only[i], do)[0], all_three[i])
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(P.window_attention(*leaves), leaves, do, create_graph=True)


def test_side_stream_and_graph():
    """On another stream than torch's default, and captured: replays with eager work between give the eager bits for new inputs."""
    q, k, v, _ = inputs(2, 1, 3000, 8, 2, 64, torch.bfloat16)
    lengths = torch.tensor([3000, 1234], device=DEV)
    call = lambda: P.window_attention(q, k, v, window=2500, sinks=2, lengths=lengths, starts=lengths - 1)  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(call(), want)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(3):
        q.copy_(rnd(q.shape, 70 + i, q.dtype))
        lengths.copy_(torch.tensor([3000 - 700 * i, 5 + 900 * i], device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())


@pytest.mark.parametrize("kw,error,match", [
    (dict(window=0), ValueError, "window"), (dict(window=-3), ValueError, "window"), (dict(sinks=-1), ValueError, "sinks"),
    (dict(scale=0.0), ValueError, "scale"), (dict(scale=-1.0), ValueError, "scale"), (dict(scale=math.nan), ValueError, "scale"),
    (dict(lengths=torch.zeros(2)), RuntimeError, "lengths"), (dict(starts=[0, 0]), RuntimeError, "starts")])
def test_refusals_of_options(kw, error, match):
    q, k, v, _ = inputs(2, 5, 5, 4, 2, 32, torch.float32)
    with pytest.raises(error, match=match):
        P.window_attention(q, k, v, **kw)


def test_refusals_of_shapes():
    q, k, v, _ = inputs(2, 5, 5, 4, 2, 32, torch.float32)
    for args in ((q[0], k, v), (q, k, v[:, :4]), (q, k[:1], v[:1]), (q[:, :, :3], k, v), (q, k.bfloat16(), v), (q[..., :12], k[..., :12], v[..., :12]),
                 (rnd((2, 5, 4, 136), 1), rnd((2, 5, 4, 136), 1), rnd((2, 5, 4, 136), 1)), (q.double(), k.double(), v.double()),
                 (q, k.cpu(), v), (q[..., :4], k[..., :4], v[..., :4])):
        with pytest.raises(RuntimeError):
            P.window_attention(*args)
    for bad in (torch.zeros(3, dtype=torch.int64, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int64)):
        with pytest.raises(RuntimeError, match="lengths"):
            P.window_attention(q, k, v, lengths=bad)
