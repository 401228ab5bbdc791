"""qk_norm_rope on the GPU against a plain implementation in float64.

Tolerances are bounds of the rounding errors, computed next to the reference from the same magnitudes: U is the rounding of a
value to its storage type (half a unit of the last place), E fp32's; a sum of n terms in any order is within n E of the sum of
its terms' magnitudes. Cosines and sines are within 4 E of 1."""
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


def rnd(shape, seed, dtype=torch.float32, std=1.0, mean=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std + mean).to(dtype)


def within(out, ref, bound, what=""):
    assert out.shape == ref.shape, (what, out.shape, ref.shape)
    err = (out.double() - ref).abs()
    bad = ~(err <= bound + 1e-300)
    assert not bool(bad.any()), (what, int(bad.sum()), float((err / (bound + 1e-300)).nan_to_num(nan=9e9).max()))


def rotation(d, rot, pos, theta, interleaved):
    """(index of the partner of each element, cosines, signed sines) of shape (batch, n, 1, d): y = u cos + u[partner] sin."""
    i = torch.arange(rot // 2, device=DEV)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    partner = torch.arange(d, device=DEV)
    partner[lo], partner[hi] = hi, lo
    cos, sin = torch.ones(*pos.shape, d, device=DEV, dtype=torch.float64), torch.zeros(*pos.shape, d, device=DEV, dtype=torch.float64)
    if rot:
        angle = pos.double()[..., None] * theta ** (-2.0 * i.double() / rot)
        cos[..., lo] = cos[..., hi] = angle.cos()
        sin[..., lo], sin[..., hi] = -angle.sin(), angle.sin()
    return partner, cos[:, :, None], sin[:, :, None]


def reference(x, w, g, norm, eps, pos, theta, rot, interleaved):
    """((y, dx, dw), their bounds) in float64."""
    d, store = x.shape[-1], U[x.dtype]
    x, w, g = x.detach().double(), torch.ones(d, device=DEV, dtype=torch.float64) if w is None else w.detach().double(), g.double()
    partner, cos, sin = rotation(d, rot, pos, theta, interleaved)
    c = x - x.mean(-1, keepdim=True) if norm == "layer" else x
    rstd = torch.ones_like(x[..., :1]) if norm is None else 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    hat = c * rstd
    # relative error of rstd: its sum of squares and root; absolute error of a normalised value besides: the mean's
    off = (d + 2) * E * x.abs().mean(-1, keepdim=True) * rstd if norm == "layer" else 0.0
    hat_err = hat.abs() * (d + 12) * E + 3 * off
    u, u_err = hat * w, hat_err * w.abs() + 2 * E * (hat * w).abs()
    turn = lambda t, s: t * cos + t[..., partner] * s  # noqa: E731
    wide = lambda t, e: e * cos.abs() + e[..., partner] * sin.abs() + 8 * E * (t.abs() + t[..., partner].abs())  # noqa: E731
    y = turn(u, sin)
    y_err = wide(u, u_err) + store * y.abs()
    du = turn(g, -sin)
    du_err = wide(g, 0 * g)
    dw, dw_err = (du * hat).flatten(0, 2), (du_err * hat.abs() + du.abs() * hat_err + 2 * E * (du * hat).abs()).flatten(0, 2)
    dw_err = dw_err.sum(0) + (dw.shape[0] + 4) * E * dw.abs().sum(0)
    dw = dw.sum(0)
    cw, cw_err = du * w, du_err * w.abs() + 2 * E * (du * w).abs()
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    dot, dot_err = mean(cw * hat), mean(cw_err * hat.abs() + cw.abs() * hat_err) + (d + 2) * E * mean((cw * hat).abs())
    if norm is None:
        dot, dot_err = dot * 0, dot_err * 0
    inner, inner_err = cw - hat * dot, cw_err + hat_err * dot.abs() + hat.abs() * dot_err + 4 * E * (cw.abs() + (hat * dot).abs())
    if norm == "layer":
        inner, inner_err = inner - mean(cw), inner_err + mean(cw_err) + (d + 4) * E * mean(cw.abs())
    dx = inner * rstd
    dx_err = rstd * (inner_err + (d + 12) * E * inner.abs()) + store * dx.abs()
    return (y, dx, dw), (y_err, dx_err, dw_err)


def check(q, k, qw, kw, *, norm="rms", eps=1e-6, positions=None, theta=10000.0, rotary_dim=None, interleaved=False):
    opt = dict(norm=norm, eps=eps, positions=positions, theta=theta, rotary_dim=rotary_dim, interleaved=interleaved)
    b, n, _, d = q.shape
    pos = (torch.arange(n, device=DEV) if positions is None else positions).expand(b, n)
    given = [t for t in (q, k, qw, kw) if t is not None]
    leaves = [None if t is None else t.detach().requires_grad_() for t in (q, k, qw, kw)]
    qo, ko = P.qk_norm_rope(leaves[0], leaves[1], q_weight=leaves[2], k_weight=leaves[3], **opt)
    with torch.no_grad():
        plain = P.qk_norm_rope(q, k, q_weight=qw, k_weight=kw, **opt)
        assert torch.equal(plain[0], qo) and (ko is None or torch.equal(plain[1], ko))
    dq, dk = rnd(q.shape, 91, q.dtype), None if k is None else rnd(k.shape, 92, q.dtype)
    grads = torch.autograd.grad([t for t in (qo, ko) if t is not None], [t for t in leaves if t is not None],
                                [t for t in (dq, dk) if t is not None])
    grads = dict(zip([i for i, t in enumerate(leaves) if t is not None], grads))
    assert [grads[i].dtype for i in grads] == [t.dtype for t in given]
    for i, (x, w, g, out) in enumerate(((q, qw, dq, qo), (k, kw, dk, ko))):
        if x is None:
            assert out is None
            continue
        (y, dx, dw), (y_err, dx_err, dw_err) = reference(x, w, g, norm, eps, pos, theta, d if rotary_dim is None else rotary_dim, interleaved)
        within(out, y, y_err, ("y", i))
        within(grads[i], dx, dx_err, ("dx", i))
        if w is not None:
            within(grads[2 + i], dw, dw_err + U[w.dtype] * dw.abs(), ("dw", i))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", ["rms", "layer", None])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,n,h,kv,d,rot", [
    (1, 1, 1, 1, 2, 2), (2, 3, 2, 1, 6, 4), (1, 5, 3, 3, 8, 8), (2, 7, 4, 2, 16, 16), (1, 9, 9, 3, 40, 20), (2, 33, 5, 1, 64, 64), (1, 10, 3, 2, 72, 0),
    (1, 65, 9, 3, 80, 40), (3, 17, 6, 2, 128, 128), (1, 4, 3, 1, 130, 64), (1, 6, 2, 1, 256, 96), (1, 3, 2, 2, 512, 512), (2, 2, 1, 1, 510, 254)])
def test_matches_float64(dtype, norm, interleaved, b, n, h, kv, d, rot):
    q, k = rnd((b, n, h, d), 1, dtype, mean=0.3), rnd((b, n, kv, d), 2, dtype, std=3.0)
    qw, kw = (None, None) if norm is None else (rnd((d,), 3, std=0.3, mean=1.0), rnd((d,), 4, std=0.3, mean=1.0))
    check(q, k, qw, kw, norm=norm, rotary_dim=rot, interleaved=interleaved)


@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_absent_or_in_their_own_dtype(dtype):
    q, k, w = rnd((2, 50, 8, 64), 1, dtype), rnd((2, 50, 2, 64), 2, dtype), rnd((64,), 3, torch.bfloat16, mean=1.0)
    check(q, k, w, w.clone())
    check(q, k, w.float(), None)
    check(q, k, None, w)
    check(q, None, w, None)
    check(q, None, None, None, norm="layer")
    check(q, k, rnd((65,), 4)[1:], rnd((65,), 5)[:64])  # (a weight that begins on an odd boundary)


@pytest.mark.parametrize("dtype", DTYPES)
def test_positions(dtype):
    """Far, negative and repeated positions, of each sequence its own or shared; other bases."""
    q, k = rnd((3, 20, 4, 32), 1, dtype), rnd((3, 20, 4, 32), 2, dtype)
    far = torch.tensor([0, 1 << 20, (1 << 40) + 12345], device=DEV)[:, None] + torch.arange(20, device=DEV)
    # (a float64 angle of 2^40 radians is off by 2^-13 itself: not compared there)
    check(q[:2], k[:2], None, None, positions=far[:2])
    check(q, k, None, None, positions=-torch.arange(20, device=DEV))
    check(q, k, None, None, positions=torch.tensor([7] * 20, device=DEV), theta=1e6)
    check(q, k, None, None, theta=1.0)
    # a whole turn of every pair further on: the angle's fraction is what counts
    one = P.qk_norm_rope(q, norm=None, positions=far[2])[0]
    two = P.qk_norm_rope(q, norm=None, positions=far[2].clone())[0]
    assert torch.equal(one, two) and one.isfinite().all()
    assert torch.allclose(one.float().norm(dim=-1), q.float().norm(dim=-1), rtol=2 ** -7)


def test_rotations_compose():
    """Turning by p and then by p' is turning by p + p': at 2^62 too, where no float holds the angle."""
    q = rnd((1, 8, 2, 64), 1)
    p = torch.tensor([1, 5, 1000, (1 << 30) + 1, (1 << 52) + 3, (1 << 62) + 7, -(1 << 61), -3], device=DEV)
    once = P.qk_norm_rope(P.qk_norm_rope(q, norm=None, positions=p)[0], norm=None, positions=17 - p)[0]
    whole = P.qk_norm_rope(q, norm=None, positions=torch.full_like(p, 17))[0]
    pair = (q ** 2 + q.roll(32, -1) ** 2).sqrt().double()
    # two rotations' roundings (8 E of the pair each) and the rates', rounded to 2^-64 turns: 2^62 of them are a quarter turn off
    # either way, and cancel: the same rate is added and taken away
    within(once, whole.double(), 40 * E * pair)


def test_constant_and_zero_rows():
    """A row of zeros stays zero; a constant one is removed by the layer norm."""
    q = torch.zeros(1, 4, 2, 64, device=DEV)
    q[:, 1] = 3.0
    q[:, 2] = 1e-30
    for norm in ("rms", "layer"):
        y, _ = P.qk_norm_rope(q, norm=norm)
        assert y.isfinite().all() and not y[:, 0].any()
        if norm == "layer":
            assert not y[:, 1].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    x = rnd((2, 30, 10, 64), 1, dtype)
    w = rnd((64,), 2, mean=1.0)
    check(x[:, :, :6], x[:, :, 6:8], w, w.clone())
    y = rnd((2, 10, 30, 64), 3, dtype).transpose(1, 2)
    check(y[:, :, :6], y[:, :, 6:8], w, w.clone())
    z = rnd((2, 30, 8, 67), 4, dtype)[..., 1:65]
    check(z[:, :, :6], z[:, :, 6:], w, w.clone())
    t = rnd((2, 30, 64, 8), 5, dtype).transpose(2, 3)
    check(t[:, :, :6], t[:, :, 6:], w, w.clone())
    check(x[:, :1, :1].expand(2, 30, 6, 64), x[:, :, 6:8], w, w.clone())


def test_many_tokens_sum_in_a_fixed_order():
    q, k, w = rnd((3, 3001, 6, 64), 1, torch.bfloat16), rnd((3, 3001, 2, 64), 2, torch.bfloat16), rnd((64,), 3, mean=1.0)
    check(q, k, w, w.clone())
    leaf = w.clone().requires_grad_()
    runs = [torch.autograd.grad(P.qk_norm_rope(q, k, q_weight=leaf)[0], leaf, q)[0] for _ in range(3)]
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_one_output_unused_and_second_backward():
    q, k = rnd((2, 9, 4, 32), 1).requires_grad_(), rnd((2, 9, 2, 32), 2).requires_grad_()
    w = rnd((32,), 3, mean=1.0).requires_grad_()
    qo, ko = P.qk_norm_rope(q, k, q_weight=w, k_weight=w)
    g = rnd(qo.shape, 4)
    a = torch.autograd.grad(qo, (q, k, w), g, retain_graph=True, allow_unused=True)
    assert a[1] is None or not a[1].any()
    b = torch.autograd.grad((qo, ko), (q, k, w), (g, torch.zeros_like(ko)), retain_graph=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2]) and not b[1].any()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(qo, q, g, create_graph=True)


def test_empty_sizes_and_graph():
    q, k, w = rnd((2, 0, 4, 32), 1).requires_grad_(), rnd((2, 0, 2, 32), 2).requires_grad_(), rnd((32,), 3).requires_grad_()
    qo, ko = P.qk_norm_rope(q, k, q_weight=w)
    assert qo.shape == q.shape and ko.shape == k.shape
    assert not torch.autograd.grad(qo.sum() + ko.sum(), (w,))[0].any()
    x, pos = rnd((4, 1, 10, 128), 4, torch.bfloat16), torch.tensor([[5], [900], [1 << 20], [0]], device=DEV)
    call = lambda: P.qk_norm_rope(x[:, :, :8], x[:, :, 8:], positions=pos)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call()
    for i in range(3):
        x.copy_(rnd(x.shape, 60 + i, x.dtype))
        pos += 1
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, call()))


@pytest.mark.parametrize("kw,error", [
    (dict(norm="batch"), ValueError), (dict(norm=None, q_weight=1), ValueError), (dict(rotary_dim=3), ValueError), (dict(rotary_dim=34), ValueError),
    (dict(rotary_dim=-2), ValueError), (dict(theta=0.5), ValueError), (dict(theta=math.inf), ValueError), (dict(eps=-1.0), ValueError),
    (dict(positions=torch.zeros(5)), RuntimeError), (dict(q_weight=2), RuntimeError)])
def test_refusals_of_options(kw, error):
    q, k = rnd((2, 5, 4, 32), 1), rnd((2, 5, 2, 32), 2)
    kw = dict(kw)
    if kw.get("q_weight"):
        kw["q_weight"] = torch.ones(32 if kw["q_weight"] == 1 else 31, device=DEV)
    with pytest.raises(error):
        P.qk_norm_rope(q, k, **kw)


def test_refusals_of_shapes():
    q, k = rnd((2, 5, 4, 32), 1), rnd((2, 5, 2, 32), 2)
    one = torch.ones(32, device=DEV)
    for args, kw in (((q[0],), {}), ((q, k[:, :4]), {}), ((q, k[..., :16]), {}), ((q, k.bfloat16()), {}), ((q[..., :31],), {}), ((q.double(),), {}),
                     ((q, k.cpu()), {}), ((rnd((1, 1, 1, 514), 1),), {}), ((q[:, :, :0],), {}),
                     ((q, k), dict(q_weight=one, k_weight=one.bfloat16())), ((q,), dict(positions=torch.zeros(6, dtype=torch.int64, device=DEV)))):
        with pytest.raises(RuntimeError):
            P.qk_norm_rope(*args, **kw)
    with pytest.raises(ValueError, match="needs k"):
        P.qk_norm_rope(q, k_weight=one)
