"""The training operators on the GPU against plain implementations in float64.

Tolerances are bounds of the rounding errors, computed next to each reference from the same magnitudes: U is the rounding
of a result to its storage type (half a unit of the last place), E fp32's; a sum of n terms in any order is within n E of
the sum of its terms' magnitudes. ETA is added where exponentials underflow."""
import math

import pytest
import torch

import psgd_pro_amd as P
from philox_ref import philox4x32_10

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -24
ETA = 2.0 ** -126  # below fp32's smallest normal a value may be 0
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


# -- dropout ----------------------------------------------------------------------------------------------------------


def mask_ref(rows, d, p, seed, stream):
    """Kept elements from the Python-integer generator."""
    per, thr = (d + 7) // 8, round(65536 * p)
    out = torch.zeros(rows, per * 8, dtype=torch.bool)
    for i in range(rows):
        for b in range(per):
            n = i * per + b
            w = philox4x32_10((n & 0xFFFFFFFF, n >> 32, stream & 0xFFFFFFFF, stream >> 32),
                              (seed & 0xFFFFFFFF, seed >> 32))
            for c in range(8):
                out[i, 8 * b + c] = ((w[c // 2] >> (16 * (c % 2))) & 0xFFFF) >= thr
    return out[:, :d].to(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d,p", [(1, 1, 0.5), (3, 7, 0.25), (2, 8, 0.1), (5, 77, 0.9), (17, 130, 0.3), (4, 513, 0.01)])
def test_dropout_matches_the_generator(dtype, rows, d, p):
    seed, stream = 0x123456789ABCDEF, (7 << 32) | 3
    x, g = rnd((rows, d), 1, dtype).requires_grad_(), rnd((rows, d), 2, dtype)
    keep, scale = mask_ref(rows, d, p, seed, stream), 65536 / (65536 - round(65536 * p))
    y = P.dropout(x, p, seed=seed, stream=stream)
    dx, = torch.autograd.grad(y, x, g)
    for out, src in ((y, x), (dx, g)):
        ref = torch.where(keep, src.detach().double() * scale, 0.0)
        within(out, ref, (U[dtype] + 2 * E) * ref.abs())
        assert torch.equal(out == 0, ~keep | (src == 0))


def test_dropout_limits_layouts_and_infinities():
    x = rnd((6, 40), 3)
    assert torch.equal(P.dropout(x, 0.0, seed=1), x)
    assert torch.equal(P.dropout(x, 1.0, seed=1), torch.zeros_like(x))
    full = P.dropout(x, 0.5, seed=5)
    wide = torch.empty(6, 64, device=DEV)
    wide[:, :40] = x
    assert torch.equal(P.dropout(wide[:, :40], 0.5, seed=5), full)       # row stride over d
    assert torch.equal(P.dropout(x.t().contiguous().t(), 0.5, seed=5), full)  # columns contiguous
    assert torch.equal(P.dropout(x.view(2, 3, 40), 0.5, seed=5).view(6, 40), full)
    assert torch.equal(P.dropout(x[0:1].expand(6, 40), 0.5, seed=5), P.dropout(x[0:1].repeat(6, 1), 0.5, seed=5))
    assert not torch.equal(P.dropout(x, 0.5, seed=5, stream=1), full) and not torch.equal(P.dropout(x, 0.5, seed=6), full)
    inf = torch.full((6, 40), math.inf, device=DEV)
    assert torch.equal(torch.isinf(P.dropout(inf, 0.5, seed=5)), full != 0)
    assert not torch.isnan(P.dropout(inf, 0.5, seed=5)).any()
    assert P.dropout(torch.empty(0, 8, device=DEV), 0.5, seed=1).shape == (0, 8)
    assert P.dropout(torch.empty(3, 0, device=DEV), 0.5, seed=1).shape == (3, 0)
    torch.manual_seed(11)
    a = P.dropout(x, 0.5)
    torch.manual_seed(11)
    assert torch.equal(P.dropout(x, 0.5), a) and not torch.equal(P.dropout(x, 0.5), a)


def test_dropout_rate_of_a_large_tensor():
    """16.7 million draws: the kept share within 6 standard deviations, and no two rows' masks alike."""
    y = P.dropout(torch.ones(4096, 4096, device=DEV, dtype=torch.bfloat16), 0.1, seed=42)
    n, q = y.numel(), round(6553.6) / 65536
    assert abs(int((y == 0).sum()) - n * q) < 6 * math.sqrt(n * q * (1 - q))
    assert torch.unique((y[:64, :256] == 0).float(), dim=0).shape[0] == 64


# -- residual_norm ----------------------------------------------------------------------------------------------------


def res_ref(x, f, par, pre, post, gate, scale, eps, keep, dy, dh, u):
    """Outputs and gradients in float64 with bounds of their errors: name -> (value, bound). u: the rounding of the
    stored results."""
    d = x.shape[1]
    K = (d + 64) * E  # sums over a row in any order, and the handful of operations around them
    xx, ff = x.double(), f.double()

    def stats(v, kind):
        mean = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
        return mean, ((v - mean).square().mean(1, keepdim=True) + eps).rsqrt()

    def w(k, fill):
        return par[k].double() if par.get(k) is not None else torch.full((d,), float(fill), device=DEV, dtype=torch.float64)

    one = torch.ones_like(xx)
    g = gate.double() if gate is not None else one
    if post:
        fm, fr = stats(ff, post)
        fh = (ff - fm) * fr
        ub = fh * w("post_weight", 1) + w("post_bias", 0)
        ub_err = K * ((ff.abs() + ff.abs().mean(1, keepdim=True)) * fr * w("post_weight", 1).abs() * 2 + w("post_bias", 0).abs() + ub.abs())
        fh_err = K * 2 * (ff.abs() + ff.abs().mean(1, keepdim=True)) * fr
    else:
        fm, fr, fh, ub, ub_err, fh_err = 0 * one, one, ff, ff, 0 * one, 0 * one
    b = ub * keep
    y = xx + scale * g * b
    y_err = (scale * g * keep).abs() * ub_err + 8 * E * (xx.abs() + (scale * g * b).abs())
    out = {"y": (y, y_err + u * y.abs())}
    m, r = stats(y, pre) if pre else (0 * one[:, :1], one[:, :1])
    hat = (y - m) * r
    hat_err = r * (y_err + y_err.mean(1, keepdim=True)) * 2 + K * 2 * (y.abs() + y.abs().mean(1, keepdim=True)) * r
    hat_err = hat_err + hat.abs() * (hat.abs() * hat_err).mean(1, keepdim=True)
    if pre:
        h = hat * w("pre_weight", 1) + w("pre_bias", 0)
        out["h"] = (h, hat_err * w("pre_weight", 1).abs() + 4 * E * (h.abs() + w("pre_bias", 0).abs()) + u * h.abs())
    if dy is None and dh is None:
        return out
    n = x.shape[0]
    dyt = dy.double() if dy is not None else 0 * one
    dyt_err = 0 * one
    if dh is not None:
        hb = hat_err
        c = dh.double() * w("pre_weight", 1)
        c1 = c.mean(1, keepdim=True) if pre == "layer" else 0
        c2 = (c * hat).mean(1, keepdim=True)
        mag = c.abs() + c.abs().mean(1, keepdim=True) + hat.abs() * (c * hat).abs().mean(1, keepdim=True)
        dyt_err = r * (hb * c2.abs() + hat.abs() * (c.abs() * hb).mean(1, keepdim=True) + 2 * K * mag) + 4 * E * dyt.abs()
        dyt_err = dyt_err + r * mag * (hat.abs() * hb).mean(1, keepdim=True)  # 1 / std's own error
        dyt = dyt + r * (c - c1 - hat * c2)
        s = (n + 8) * E
        out["pre_weight"] = ((dh.double() * hat).sum(0), (dh.double().abs() * (hb + s * hat.abs())).sum(0))
        out["pre_bias"] = (dh.double().sum(0), s * dh.double().abs().sum(0))
    out["x"] = (dyt, dyt_err + u * dyt.abs())
    du = scale * g * keep * dyt
    du_err = (scale * g * keep).abs() * (dyt_err + 4 * E * dyt.abs())
    s = (n + 8) * E
    dg = scale * dyt * b
    out["gate"] = (dg, abs(scale) * (dyt_err * b.abs() + dyt.abs() * keep * ub_err + s * (dyt * b).abs()))
    if post:
        out["post_weight"] = ((du * fh).sum(0), (du_err * fh.abs() + du.abs() * (fh_err + s * fh.abs())).sum(0))
        out["post_bias"] = (du.sum(0), (du_err + s * du.abs()).sum(0))
        c, c_err = du * w("post_weight", 1), du_err * w("post_weight", 1).abs()
        c1 = c.mean(1, keepdim=True) if post == "layer" else 0
        c2 = (c * fh).mean(1, keepdim=True)
        mag = c.abs() + c.abs().mean(1, keepdim=True) + fh.abs() * (c * fh).abs().mean(1, keepdim=True)
        df = fr * (c - c1 - fh * c2)
        df_err = fr * (c_err + c_err.mean(1, keepdim=True) + fh.abs() * (c_err * fh.abs() + c.abs() * fh_err).mean(1, keepdim=True)
                       + fh_err * c2.abs() + 2 * K * mag)
        df_err = df_err + fr * mag * (fh.abs() * fh_err).mean(1, keepdim=True)
    else:
        df, df_err = du, du_err
    out["f"] = (df, df_err + u * df.abs())
    return out


def run_res(shape, dtype, pre, post, gate_shape, p=0.0, affine=True, wdtype=torch.float32, scale=0.75, eps=1e-5, use=("dy", "dh"),
            layout=lambda t: t, gate_dtype=None):
    d = shape[-1]
    n = math.prod(shape[:-1])
    x, f = rnd(shape, 1, dtype, 1.5, 0.2), rnd(shape, 2, dtype, 0.7, -0.1)
    par = {}
    if affine:
        if pre:
            par["pre_weight"] = rnd(d, 3, wdtype, 0.2, 1.0)
        if pre == "layer":
            par["pre_bias"] = rnd(d, 4, wdtype, 0.3)
        if post:
            par["post_weight"] = rnd(d, 5, wdtype, 0.2, 1.0)
        if post == "layer":
            par["post_bias"] = rnd(d, 6, wdtype, 0.3)
    gate = None if gate_shape is None else rnd(gate_shape, 7, gate_dtype or dtype, 0.5, 0.5)
    dy, dh = rnd(shape, 8, dtype), rnd(shape, 9, dtype)
    leaves = {"x": layout(x).requires_grad_(), "f": layout(f).requires_grad_(), **{k: v.requires_grad_() for k, v in par.items()}}
    if gate is not None:
        leaves["gate"] = gate.requires_grad_()
    y, h = P.residual_norm(leaves["x"], leaves["f"], pre=pre, post=post, gate=leaves.get("gate"), scale=scale, eps=eps, p=p,
                           seed=99, stream=4, **{k: leaves[k] for k in par})
    keep = torch.ones(n, d, device=DEV, dtype=torch.float64)
    if p:
        keep = P.dropout(torch.ones(n, d, device=DEV), p, seed=99, stream=4).double()
    gd = None
    if gate is not None:
        gd = gate.detach().expand(shape).reshape(n, d)
    use_y, use_h = "dy" in use, "dh" in use and pre is not None
    ref = res_ref(x.detach().reshape(n, d), f.detach().reshape(n, d), {k: v.detach() for k, v in par.items()}, pre, post, gd, scale,
                  eps, keep, dy.reshape(n, d) if use_y else None, dh.reshape(n, d) if use_h else None, U[dtype])
    within(y.reshape(n, d), *ref["y"], "y")
    if pre:
        within(h.reshape(n, d), *ref["h"], "h")
    else:
        assert h is None
    outs, gs = zip(*[(o, g) for o, g, u in ((y, dy, use_y), (h, dh, use_h)) if u])
    names = [k for k in leaves if use_h or not k.startswith("pre")]
    grads = dict(zip(names, torch.autograd.grad(outs, [leaves[k] for k in names], gs)))
    for k, g in grads.items():
        v, b = ref[k]
        if k == "gate":
            v, b = v.view(shape).sum_to_size(gate.shape), b.view(shape).sum_to_size(gate.shape)
            b = b + U[gate.dtype] * v.abs()
            g, v, b = (t.reshape(-1, d) for t in (g, v, b))
        elif k.endswith(("weight", "bias")):
            b = b + U[wdtype] * v.abs()
        else:
            g = g.reshape(n, d)
        assert g.dtype == leaves[k].dtype
        within(g, v, b, k)
    with torch.no_grad():  # without gradients the same values
        y2, h2 = P.residual_norm(x, f, pre=pre, post=post, gate=gate, scale=scale, eps=eps, p=p, seed=99, stream=4, **par)
    assert torch.equal(y, y2) and (h is None or torch.equal(h, h2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pre,post", [("rms", None), ("rms", "rms"), ("layer", None), ("layer", "layer"), (None, "rms"),
                                      ("rms", "layer")])
@pytest.mark.parametrize("d", [1, 7, 8, 63, 512, 513, 770, 1025, 2304, 4096])
def test_residual_norm_sizes(dtype, pre, post, d):
    run_res((5, d), dtype, pre, post, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [4104, 8192, 8200, 16384 + 3])
@pytest.mark.parametrize("post,gate", [("rms", "seq"), (None, "channel")])
def test_residual_norm_long_rows(dtype, d, post, gate):
    run_res((2, 3, d), dtype, "layer", post, (2, 1, d) if gate == "seq" else (d,), p=0.1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [2047, 4097, 4101, 6962, 8191])
@pytest.mark.parametrize("pre,post,gate", [("rms", None, None), ("rms", "rms", None), ("rms", None, "token"), ("layer", None, None),
                                           ("rms", "rms", "seq"), ("layer", "rms", None), ("layer", "layer", "token")])
def test_residual_norm_long_rows_that_end_inside_a_vector(dtype, d, pre, post, gate):
    shape = {None: None, "seq": (2, 1, d), "token": (2, 5, d)}[gate]
    run_res((2, 5, d), dtype, pre, post, shape, p=0.1 if d % 3 else 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", ["channel", "ones", "seq", "token"])
@pytest.mark.parametrize("batch,tokens,d", [(1, 1, 64), (3, 1, 72), (5, 9, 130), (2, 700, 96), (700, 2, 520), (3, 65, 1100)])
def test_residual_norm_gates(dtype, gate, batch, tokens, d):
    shape = {"channel": (d,), "ones": (1, 1, d), "seq": (batch, 1, d), "token": (batch, tokens, d)}[gate]
    run_res((batch, tokens, d), dtype, "rms", "layer" if tokens == 9 else None, shape, p=0.25 if d > 100 else 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wdtype", DTYPES)
def test_residual_norm_parameter_types(dtype, wdtype):
    run_res((4, 33, 200), dtype, "layer", "rms", (4, 1, 200), wdtype=wdtype, gate_dtype=wdtype)
    run_res((4, 33, 200), dtype, "layer", "layer", None, affine=False)


@pytest.mark.parametrize("use", [("dy",), ("dh",)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_residual_norm_one_gradient_only(dtype, use):
    run_res((6, 300), dtype, "rms", "rms", (300,), use=use)


@pytest.mark.parametrize("dtype", DTYPES)
def test_residual_norm_layouts(dtype):
    def strided(t):
        w = torch.zeros(*t.shape[:-1], t.shape[-1] + 5, device=DEV, dtype=t.dtype)
        w[..., :t.shape[-1]] = t
        return w[..., :t.shape[-1]].detach()

    run_res((7, 264), dtype, "rms", "rms", None, layout=strided)
    run_res((3, 5, 264), dtype, "layer", None, (3, 1, 264), layout=lambda t: t.transpose(0, 1).contiguous().transpose(0, 1))
    run_res((7, 264), dtype, "rms", None, None, layout=lambda t: t.t().contiguous().t())


def test_residual_norm_many_rows_and_shared_weights_are_deterministic():
    x, f = rnd((5000, 256), 1, torch.bfloat16).requires_grad_(), rnd((5000, 256), 2, torch.bfloat16).requires_grad_()
    w = rnd(256, 3, mean=1.0).requires_grad_()
    g = rnd((5000, 256), 4, torch.bfloat16)

    def grads():
        y, h = P.residual_norm(x, f, pre_weight=w, post="rms", post_weight=w)
        return torch.autograd.grad((y, h), (x, f, w), (g, g))

    a, b = grads(), grads()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_residual_norm_without_a_block():
    x, g = rnd((5, 96), 1).requires_grad_(), rnd((5, 96), 2)
    w = rnd(96, 3, mean=1.0).requires_grad_()
    y, h = P.residual_norm(x, pre_weight=w, eps=1e-5)
    assert torch.equal(y, x)
    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    hd = xd * (xd.square().mean(1, keepdim=True) + 1e-5).rsqrt() * wd
    within(h, hd.detach(), 200 * E * hd.detach().abs())
    for out, ref in zip(torch.autograd.grad((y, h), (x, w), (g, g)),
                        torch.autograd.grad((hd, xd * 1), (xd, wd), (g.double(), g.double()))):
        within(out, ref, 400 * E * (ref.abs().mean() + ref.abs()) * 8)


def test_residual_norm_zero_rows_constant_rows_and_empty_inputs():
    x = torch.zeros(3, 128, device=DEV)
    f = torch.zeros(3, 128, device=DEV)
    x[1], f[2] = 3.0, 3.0
    y, h = P.residual_norm(x, f, pre="layer", post="rms", eps=1e-6)
    assert torch.equal(h[0], torch.zeros(128, device=DEV)) and torch.isfinite(h).all()
    assert torch.equal(h[1], torch.zeros(128, device=DEV))  # a constant row has no deviation
    e = torch.empty(0, 128, device=DEV, requires_grad=True)
    w = torch.ones(128, device=DEV, requires_grad=True)
    y, h = P.residual_norm(e, e, pre_weight=w)
    assert y.shape == h.shape == (0, 128)
    assert torch.equal(torch.autograd.grad(h.sum(), w)[0], torch.zeros(128, device=DEV))


def test_residual_norm_gradient_against_differences():
    """Central differences of the operator itself along a direction; the difference's own truncation is taken from the
    float64 formula at the same step."""
    shape, d, step = (6, 80), 80, 2.0 ** -7
    x, f, dirx, dirf = (rnd(shape, k) for k in (1, 2, 3, 4))
    gy, gh = rnd(shape, 5).double(), rnd(shape, 6).double()

    def value(a, b):
        y, h = P.residual_norm(a, b, pre="layer", post="rms", scale=0.5, eps=1e-5)
        return float((y.double() * gy).sum() + (h.double() * gh).sum())

    def plain(a, b):
        u = b * (b.square().mean(1, keepdim=True) + 1e-5).rsqrt()
        y = a + 0.5 * u
        c = y - y.mean(1, keepdim=True)
        return float((y * gy).sum() + (c * (c.square().mean(1, keepdim=True) + 1e-5).rsqrt() * gh).sum())

    xs, fs = x.clone().requires_grad_(), f.clone().requires_grad_()
    y, h = P.residual_norm(xs, fs, pre="layer", post="rms", scale=0.5, eps=1e-5)
    gx, gf = torch.autograd.grad((y, h), (xs, fs), (gy.float(), gh.float()))
    slope = float((gx.double() * dirx.double()).sum() + (gf.double() * dirf.double()).sum())
    diff = (value(x + step * dirx, f + step * dirf) - value(x - step * dirx, f - step * dirf)) / (2 * step)
    X, F, DX, DF = (t.double() for t in (x, f, dirx, dirf))
    at = lambda s: (plain(X + s * DX, F + s * DF) - plain(X - s * DX, F - s * DF)) / (2 * s)  # noqa: E731
    trunc = abs(at(step) - at(2.0 ** -16)) + 1e-6
    noise = 64 * E * float((gy.abs() + gh.abs()).sum() * 3) / step
    assert abs(diff - slope) <= trunc + noise


def test_residual_norm_refusals():
    x = rnd((4, 6, 32), 1)
    bad = [(dict(pre="batch"), ValueError), (dict(post="rms"), ValueError), (dict(pre=None), ValueError),
           (dict(f=x[:2]), RuntimeError), (dict(f=x.bfloat16()), RuntimeError), (dict(f=x.half()), RuntimeError),
           (dict(f=x, pre_bias=x[0, 0]), ValueError), (dict(f=x, pre_weight=x[0, 0, :5]), RuntimeError),
           (dict(f=x, post_weight=x[0, 0]), ValueError), (dict(f=x, gate=rnd((6, 1, 32), 2)), RuntimeError),
           (dict(f=x, gate=rnd((1, 6, 32), 2)), RuntimeError), (dict(f=x, gate=rnd((4, 6, 31), 2)), RuntimeError),
           (dict(f=x, p=-0.1), ValueError), (dict(f=x, pre_weight=x[0, 0], post="rms", post_weight=x[0, 0].bfloat16()),
                                             RuntimeError), (dict(f=x, gate=torch.ones(32)), RuntimeError)]
    for kw, exc in bad:
        with pytest.raises(exc):
            P.residual_norm(x, **kw)
    with pytest.raises(RuntimeError):
        P.residual_norm(torch.zeros(4, 8, device=DEV, dtype=torch.int32))
    with pytest.raises(ValueError):
        P.dropout(x, 1.5)


# -- linear_cross_entropy -----------------------------------------------------------------------------------------------


def lce_ref(x, w, t, ignore, weight):
    """Losses and gradients of sum_i weight_i loss_i in float64, with bounds. A logit is within Z of its value: d products
    summed in any order in fp32 (products of bf16 are exact there). A softmax entry then moves by a factor within
    exp(2 Z); the operator keeps it, or the exponential it is made of, and the weighted row each in the storage type on
    the bf16 path (U) before the sums over the vocabulary and over the rows."""
    n, d = x.shape
    v = w.shape[0]
    u = U[x.dtype]
    X, W = x.double(), w.double()
    ok = t != ignore
    X = torch.where(ok[:, None], X, 0.0)
    z = X @ W.t()
    zmag = X.abs() @ W.abs().t()
    zerr = ((d + 64) * E * zmag).amax(1)
    tt = torch.where(ok, t, 0)
    lse = torch.logsumexp(z, 1)
    zt = z.gather(1, tt[:, None]).squeeze(1)
    loss = torch.where(ok, lse - zt, 0.0)
    loss_err = torch.where(ok, v * ETA + 2 * zerr + (v + 64) * E * (1 + loss.abs()) + 4 * E * (zt.abs() + lse.abs()), 0.0)
    p = torch.exp(z - lse[:, None])
    rest = p.clone().scatter_(1, tt[:, None], 0.0).sum(1)
    dz = p.scatter(1, tt[:, None], -rest[:, None]) * (weight * ok)[:, None]
    rel = 4 * zerr + (0 if x.dtype == torch.float32 else 2 * u) + (v + 128) * E
    dx = dz @ W
    dx_err = (dz.abs() @ W.abs()) * (rel + (v + 64) * E)[:, None] + u * dx.abs() + v * ETA * W.abs().sum(0)
    dw = dz.t() @ X
    dw_err = dz.abs().t() @ (X.abs() * (rel + (n + 64) * E)[:, None]) + u * dw.abs() + v * ETA * X.abs().sum(0)
    return (loss, loss_err), (dx, dx_err), (dw, dw_err)


def targets(n, v, seed, ignored=0.0, ignore=-100):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = torch.randint(v, (n,), generator=g, device=DEV)
    if n > 2:
        t[0], t[1] = v - 1, 0
    return t.masked_fill(torch.rand(n, generator=g, device=DEV) < ignored, ignore)


def run_lce(x, w, t, ignore=-100, reductions=("mean", "sum", "none")):
    n = t.numel()
    count = max(1, int((t != ignore).sum()))
    gw = torch.rand(n, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)) + 0.5
    with torch.no_grad():
        plain = P.linear_cross_entropy(x, w, t, ignore_index=ignore, reduction="none")
    for red in reductions:
        weight = {"mean": torch.full((n,), 1.0 / count, device=DEV), "sum": torch.ones(n, device=DEV), "none": gw}[red].double()
        (loss, le), (dx, dxe), (dw, dwe) = lce_ref(x.detach(), w.detach(), t, ignore, weight)
        within(plain, loss, le, "loss without gradients")
        xs, ws = x.detach().requires_grad_(), w.detach().requires_grad_()
        out = P.linear_cross_entropy(xs, ws, t, ignore_index=ignore, reduction=red)
        assert out.dtype == torch.float32
        if red == "none":
            within(out, loss, le, "loss")
            gx, gw_ = torch.autograd.grad(out, (xs, ws), gw)
        else:
            within(out.detach().view(1), (loss * weight).sum().view(1), ((le + (n + 8) * E * loss) * weight).sum(), red)
            scale = 1.0 if red == "mean" else 3.0
            gx, gw_ = torch.autograd.grad(out * scale, (xs, ws))
            extra = 0.0 if scale == 1.0 else U[x.dtype]  # the gradient's scale is applied to the stored gradient
            dx, dxe, dw, dwe = dx * scale, dxe * scale + extra * (dx * scale).abs() * 1.01, dw * scale, dwe * scale + extra * (dw * scale).abs() * 1.01
        assert gx.dtype == x.dtype and gw_.dtype == w.dtype
        within(gx, dx, dxe, red + " dx")
        within(gw_, dw, dwe, red + " dw")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,v", [(1, 8, 1), (1, 1, 2), (2, 64, 1000), (3, 770, 1001), (17, 33, 130), (65, 96, 257), (129, 512, 4099),
                                   (300, 256, 513), (257, 264, 255), (512, 128, 2048), (16, 1024, 32768), (700, 72, 300)])
def test_cross_entropy_sizes(dtype, n, d, v):
    x, w = rnd((n, d), 1, dtype), rnd((v, d), 2, dtype, 1.5 / math.sqrt(d))
    run_lce(x, w, targets(n, v, 3, 0.2))


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_parts_of_a_long_vocabulary(dtype):
    """dx of few rows adds up many parts of the vocabulary: their lengths do not divide it (the last ones short, or not
    there), with more output tiles than one a CU and with fewer."""
    for n, d, v in ((64, 256, 16400), (300, 1000, 16447), (1100, 520, 33000)):
        run_lce(rnd((n, d), 1, dtype), rnd((v, d), 2, dtype, 1.5 / math.sqrt(d)), targets(n, v, 3, 0.2), reductions=("mean",))


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_everything_ignored(dtype):
    x, w = rnd((40, 64), 1, dtype).requires_grad_(), rnd((300, 64), 2, dtype).requires_grad_()
    t = torch.full((40,), 7, device=DEV)
    for red in ("mean", "sum"):
        out = P.linear_cross_entropy(x, w, t, ignore_index=7, reduction=red)
        assert float(out) == 0.0
        for g in torch.autograd.grad(out, (x, w)):
            assert torch.equal(g, torch.zeros_like(g))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 5, 40, 300])
def test_cross_entropy_ignored_rows_hold_anything(dtype, n):
    """Infinities and NaN in the ignored rows of x reach nothing; other rows' results do not change with them."""
    x, w, t = rnd((n, 96), 1, dtype), rnd((777, 96), 2, dtype, 0.2), targets(n, 777, 3)
    t[::2] = -100
    a = x.clone()
    a[0::4], a[2::4] = math.nan, math.inf
    res = []
    for q in (x, a):
        q = q.detach().requires_grad_()
        ws = w.detach().requires_grad_()
        out = P.linear_cross_entropy(q, ws, t)
        res.append((out.detach(), *torch.autograd.grad(out, (q, ws)), P.linear_cross_entropy(q.detach(), w, t, reduction="none")))
    for p, q in zip(*res):
        assert torch.equal(p, q)
    assert torch.equal(res[0][1][::2], torch.zeros_like(x[::2])) and float(res[0][3][::2].abs().sum()) == 0


@pytest.mark.parametrize("n", [1, 16, 17, 32, 33, 64, 65])
@pytest.mark.parametrize("d,v", [(40, 24576), (72, 24575), (33, 49152), (136, 49151), (256, 50001)])
def test_cross_entropy_losses_of_a_few_rows(n, d, v):
    x, w = rnd((n, d), 51, torch.bfloat16), rnd((v, d), 52, torch.bfloat16, 1.5 / math.sqrt(d))
    t = targets(n, v, 53, 0.2)
    (loss, err), _, _ = lce_ref(x, w, t, -100, torch.ones(n, device=DEV, dtype=torch.float64))
    within(P.linear_cross_entropy(x, w, t, reduction="none"), loss, err)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pattern", ["prompt", "padding", "alternate", "one", "first", "last"])
@pytest.mark.parametrize("n,d,v", [(700, 72, 600), (4500, 24, 130), (65, 40, 300)])
def test_cross_entropy_patterns_of_ignored_rows(dtype, pattern, n, d, v):
    """Rows that count are gathered: whichever they are, each loss and gradient lies at its own row, the others are 0."""
    i = torch.arange(n, device=DEV)
    keep = {"prompt": i % 97 >= 50, "padding": i < n * 2 // 3, "alternate": i % 2 == 1, "one": i == n // 2, "first": i == 0,
            "last": i == n - 1}[pattern]
    x, w = rnd((n, d), 31, dtype).requires_grad_(), rnd((v, d), 32, dtype, std=0.3).requires_grad_()
    t = targets(n, v, 33).masked_fill(~keep, -100)
    run_lce(x, w, t)
    loss = P.linear_cross_entropy(x, w, t, reduction="none")
    dx, = torch.autograd.grad(loss.sum(), x)
    assert torch.equal(loss[~keep], torch.zeros_like(loss[~keep])) and torch.equal(dx[~keep], torch.zeros_like(dx[~keep]))
    kept = int(keep.sum())
    if dtype == torch.bfloat16 and (n > 512) == (kept > 512):  # the same bits as from the others alone (the same kernels)
        xs = x.detach()[keep].requires_grad_()
        alone = P.linear_cross_entropy(xs, w, t[keep], reduction="none")
        if kept > 64:  # (up to 64 rows take a kernel of their own where there are no gradients)
            assert torch.equal(alone, loss[keep])
        assert torch.equal(torch.autograd.grad(alone.sum(), xs)[0], dx[keep])


# Up to 512 rows and 2^23 logits have kernels of their own: both sides of each limit, and what the smaller tests look at once
# more with more rows.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,v", [(511, 40, 700), (512, 96, 257), (513, 96, 257), (512, 24, 16384), (512, 24, 16385), (2, 16, 4194304),
                                   (3, 16, 4194304), (1500, 33, 4095), (1500, 64, 4096)])
def test_cross_entropy_sizes_at_the_limits(dtype, n, d, v):
    if v > 1 << 20 and dtype == torch.float32:
        v //= 4
    x, w = rnd((n, d), 61, dtype), rnd((v, d), 62, dtype, 1.5 / math.sqrt(d))
    run_lce(x, w, targets(n, v, 63, 0.2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gain", [1e-3, 30.0, 300.0])
@pytest.mark.parametrize("n", [520, 1030])
def test_cross_entropy_many_sharp_and_flat_rows(dtype, gain, n):
    d, v = 64, 1500
    w = rnd((v, d), 2, dtype, 1.0 / math.sqrt(d))
    t = targets(n, v, 3)
    x = rnd((n, d), 1, dtype)
    x[::3] = (w[t[::3]].float() * 8 / w[t[::3]].float().square().sum(1, keepdim=True)).to(dtype)
    x[1::3] = -x[1::3]
    run_lce((x.float() * gain).to(dtype), w, t, reductions=("mean", "none"))


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_many_rows_in_other_layouts(dtype):
    n = 700
    x, w, t = rnd((n, 200), 1, dtype), rnd((530, 200), 2, dtype, 0.1), targets(n, 530, 3, 0.3)

    def padded(q, pad):
        b = torch.full((q.shape[0], q.shape[1] + pad), math.nan, device=DEV, dtype=q.dtype)
        b[:, :q.shape[1]] = q
        return b[:, :q.shape[1]]

    for xs, ws in ((padded(x, 8), padded(w, 24)), (padded(x, 3), padded(w, 1)), (x.t().contiguous().t(), w.t().contiguous().t())):
        run_lce(xs, ws, t, reductions=("mean",))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [40, 700])
def test_cross_entropy_foreign_targets_stay_in_their_rows(dtype, n):
    """A target outside the vocabulary makes its own loss and dx NaN, no other row's, and dw."""
    x, w = rnd((n, 32), 1, dtype).requires_grad_(), rnd((50, 32), 2, dtype).requires_grad_()
    t = targets(n, 50, 3)
    t[3], t[n // 2], t[5] = 50, -1, -100
    foreign = torch.zeros(n, dtype=torch.bool, device=DEV)
    foreign[3] = foreign[n // 2] = True
    loss = P.linear_cross_entropy(x, w, t, reduction="none")
    assert torch.equal(torch.isnan(loss), foreign)
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    assert torch.equal(torch.isnan(dx).all(1), foreign) and torch.equal(torch.isnan(dx).any(1), foreign)
    assert torch.isnan(dw).all() and not dx[5].any()


@pytest.mark.parametrize("kept", [1, 700, 6000])
@pytest.mark.parametrize("d,v", [(40, 200), (136, 1000)])
def test_cross_entropy_parts_of_many_rows(kept, d, v):
    """dw of a small vocabulary adds up parts of the rows; where few of them count the last parts are empty."""
    n = 6000
    x, w = rnd((n, d), 71, torch.bfloat16), rnd((v, d), 72, torch.bfloat16, 1.0 / math.sqrt(d))
    t = targets(n, v, 73)
    t[kept:] = -100
    run_lce(x, w, t)


@pytest.mark.parametrize("n,d,v", [(6001, 40, 200), (3000, 136, 1000), (1025, 256, 130), (2050, 33, 260)])
def test_cross_entropy_parts_of_many_rows_in_float32(n, d, v):
    x, w = rnd((n, d), 81), rnd((v, d), 82, std=1.0 / math.sqrt(d))
    run_lce(x, w, targets(n, v, 83, 0.1))


def test_cross_entropy_slabs_without_a_row_that_counts():
    """More rows than the logits' memory holds at once: what counts fills the first slabs only."""
    n, d, v = 12000, 8, 50021
    x, w = rnd((n, d), 41, torch.bfloat16).requires_grad_(), rnd((v, d), 42, torch.bfloat16, std=0.3).requires_grad_()
    for kept in (0, 300, 11000):
        t = targets(n, v, 43)
        t[:n - kept] = -100  # the last `kept` rows
        loss = P.linear_cross_entropy(x, w, t, reduction="sum")
        dx, dw = torch.autograd.grad(loss, (x, w))
        xs = x.detach()[n - kept:].requires_grad_()
        if kept:
            some = P.linear_cross_entropy(xs, w, t[n - kept:], reduction="sum")
            sx, sw = torch.autograd.grad(some, (xs, w))
            # the same slabs either way; a single one sums the vocabulary in other parts (rows of softmax - 1: sum below 2)
            if kept == 11000:
                assert torch.equal(dx[n - kept:], sx)
            else:
                within(dx[n - kept:], sx.double(), 2 * U[torch.bfloat16] * sx.double().abs() + (v + 64) * E * 2 * w.abs().max())
            assert torch.equal(dw, sw)
            assert abs(float(loss) - float(some)) <= n * E * float(some)
        else:
            assert float(loss) == 0 and not dw.any()
        assert not dx[:n - kept].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gain", [1e-3, 30.0, 300.0])
def test_cross_entropy_sharp_and_flat_rows(dtype, gain):
    """Logits from nearly equal to a spread of a thousand: rows sure of their target (the loss underflows to zero
    smoothly), and rows whose target lies hundreds of nats below the maximum."""
    n, d, v = 96, 64, 1500
    w = rnd((v, d), 2, dtype, 1.0 / math.sqrt(d))
    t = targets(n, v, 3)
    x = rnd((n, d), 1, dtype)
    x[::3] = (w[t[::3]].float() * 8 / w[t[::3]].float().square().sum(1, keepdim=True)).to(dtype)
    x[1::3] = -x[1::3]
    run_lce((x.float() * gain).to(dtype), w, t, reductions=("mean", "none"))


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_layouts(dtype):
    x, w, t = rnd((6, 11, 200), 1, dtype), rnd((530, 200), 2, dtype, 0.1), targets(66, 530, 3, 0.3)
    ref = P.linear_cross_entropy(x, w, t.view(6, 11), reduction="none")
    assert ref.shape == (6, 11)

    def padded(q, pad):
        b = torch.full((q.shape[0], q.shape[1] + pad), math.nan, device=DEV, dtype=q.dtype)
        b[:, :q.shape[1]] = q
        return b[:, :q.shape[1]]

    x2 = x.view(66, 200)
    for xs, ws in ((padded(x2, 8), padded(w, 24)), (padded(x2, 3), padded(w, 1)), (x2.t().contiguous().t(), w.t().contiguous().t())):
        run_lce(xs, ws, t, reductions=("mean",))
    # rows that start off any 4-byte boundary
    flat = torch.empty(66 * 201 + 1, device=DEV, dtype=dtype)
    odd = flat[1:].as_strided((66, 200), (201, 1))
    odd.copy_(x2)
    run_lce(odd, w, t, reductions=("mean",))


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_foreign_targets_are_loud(dtype):
    x, w = rnd((4, 32), 1, dtype), rnd((50, 32), 2, dtype)
    loss = P.linear_cross_entropy(x, w, torch.tensor([3, 50, -1, 49], device=DEV), reduction="none")
    assert torch.equal(torch.isnan(loss), torch.tensor([False, True, True, False], device=DEV))


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_parts_of_the_gradient_and_repeated_backward(dtype):
    x, w, t = rnd((70, 64), 1, dtype), rnd((400, 64), 2, dtype, 0.2), targets(70, 400, 3, 0.1)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = P.linear_cross_entropy(xs, ws, t)
    a = [g.clone() for g in torch.autograd.grad(out * 2, (xs, ws), retain_graph=True)]
    b = torch.autograd.grad(out * 2, (xs, ws))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    only_x, = torch.autograd.grad(P.linear_cross_entropy(xs, w, t) * 2, xs)
    only_w, = torch.autograd.grad(P.linear_cross_entropy(x, ws, t) * 2, ws)
    assert torch.equal(only_x, a[0]) and torch.equal(only_w, a[1])


def test_cross_entropy_more_rows_than_a_slab():
    """More rows than the workspace holds at once, over a large vocabulary: pieces of rows add up, bit for bit the same
    in each run."""
    n, d, v = 2500, 64, 131072
    for dtype, n in ((torch.float32, 2500), (torch.bfloat16, 4500)):
        x, w = rnd((n, d), 1, dtype), rnd((v, d), 2, dtype, 0.2)
        t = targets(n, v, 3, 0.1)
        run_lce(x, w, t, reductions=("mean",))
        xs, ws = x.requires_grad_(), w.requires_grad_()
        a = torch.autograd.grad(P.linear_cross_entropy(xs, ws, t), (xs, ws))
        b = torch.autograd.grad(P.linear_cross_entropy(xs, ws, t), (xs, ws))
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_cross_entropy_gradient_against_differences():
    n, d, v, step = 9, 40, 333, 2.0 ** -7
    x, w, dx, dw = rnd((n, d), 1), rnd((v, d), 2, std=0.3), rnd((n, d), 3), rnd((v, d), 4, std=0.3)
    t = targets(n, v, 5, 0.2)
    ok = t != -100

    def plain(a, b):
        z = a.double() @ b.double().t()
        each = torch.logsumexp(z, 1) - z.gather(1, t.clamp(min=0)[:, None]).squeeze(1)
        return float(each[ok].mean())

    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(P.linear_cross_entropy(xs, ws, t), (xs, ws))
    slope = float((gx.double() * dx.double()).sum() + (gw.double() * dw.double()).sum())
    f = lambda s: float(P.linear_cross_entropy(x + s * dx, w + s * dw, t))  # noqa: E731
    X, W, DX, DW = (q.double() for q in (x, w, dx, dw))
    g = lambda s: (plain(X + s * DX, W + s * DW) - plain(X - s * DX, W - s * DW)) / (2 * s)  # noqa: E731
    trunc = abs(g(step) - g(2.0 ** -16)) + 1e-6
    noise = 2 * (d + 64) * E * float((x.abs() @ w.abs().t()).max()) * 2 / step
    assert abs((f(step) - f(-step)) / (2 * step) - slope) <= trunc + noise


def test_cross_entropy_refusals():
    x, w, t = rnd((4, 32), 1), rnd((50, 32), 2), torch.zeros(4, device=DEV, dtype=torch.int64)
    for args, exc in (((x, w.bfloat16(), t), RuntimeError), ((x.half(), w.half(), t), RuntimeError), ((x, w[:, :31], t), RuntimeError),
                      ((x, w, t.int()), RuntimeError), ((x, w, t[:3]), RuntimeError), ((x, w, t.cpu()), RuntimeError),
                      ((x, w[:0], t), RuntimeError)):
        with pytest.raises(exc):
            P.linear_cross_entropy(*args)
    with pytest.raises(ValueError):
        P.linear_cross_entropy(x, w, t, reduction="max")
    e = torch.empty(0, 32, device=DEV, requires_grad=True)
    ws = w.clone().requires_grad_()
    out = P.linear_cross_entropy(e, ws, t[:0])
    assert float(out) == 0
    assert torch.equal(torch.autograd.grad(out, ws)[0], torch.zeros_like(w))


# -- together -----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
def test_operators_on_a_side_stream(dtype):
    """The same results on another stream than the inputs' own, its work ordered behind theirs."""
    x, f, w, t = rnd((200, 256), 1, dtype), rnd((200, 256), 2, dtype), rnd((1000, 256), 3, dtype, 0.1), targets(200, 1000, 4, 0.2)

    def all_of():
        xs, fs, ws = (q.detach().requires_grad_() for q in (x, f, w))
        y, h = P.residual_norm(xs, fs, post="rms", p=0.1, seed=3)
        loss = P.linear_cross_entropy(P.dropout(h, 0.2, seed=4), ws, t) + y.float().square().mean()
        return (loss.detach(), *torch.autograd.grad(loss, (xs, fs, ws)))

    ref = all_of()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = all_of()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(ref, out))
