"""The training operators on the GPU where a step goes wrong or is unusually large: infinite logits, more rows or
gates than one launch holds workgroups for, forward passes that are run again. References in float64, bounds as in test_train_ops.py."""
import math

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import psgd_pro_amd as P
from test_train_ops import DEV, DTYPES, E, U, lce_ref, res_ref, rnd, targets, within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(hip):
    return hip


# -- logits that overflow -----------------------------------------------------------------------------------------------

BIG = 2.0 ** 100  # its square overflows float32


def overflowing(n, v, dtype, kind):
    """Every third row has an infinite logit: (x, w, targets, those rows). Column 0 of w holds BIG or -BIG at one place
    of the vocabulary and -BIG at another, column 1 -BIG everywhere, and only the rows meant have BIG in x there."""
    d = 24
    x, w, t = rnd((n, d), 91, dtype), rnd((v, d), 92, dtype, 0.3), targets(n, v, 93)
    x[:, :2], w[:, 0], w[:, 1] = 0, 0, -BIG
    hit = torch.arange(n, device=DEV) % 3 == 1
    at, other = v // 2, 3
    t = torch.where(t == at, at + 1, t)
    t[hit] = at if kind != "another +inf" else at + 1
    x[hit, 1 if kind == "all -inf" else 0] = BIG
    w[at, 0] = BIG if "+inf" in kind else -BIG
    if kind == "target and another -inf":
        w[other, 0] = -BIG
    return x, w, t, hit


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v", [(3, 70), (40, 1100), (600, 1100)])
@pytest.mark.parametrize("kind,loss_is", [("target +inf", math.nan), ("another +inf", math.nan), ("target -inf", math.inf),
                                          ("target and another -inf", math.inf), ("all -inf", math.nan)])
def test_cross_entropy_of_infinite_logits(dtype, n, v, kind, loss_is):
    """inf - inf is NaN and stays in its row, whichever kernels the sizes choose; a target of -inf costs infinitely much."""
    x, w, t, hit = overflowing(n, v, dtype, kind)

    def check(loss, what):
        got = loss[hit]
        assert bool((torch.isnan(got) if math.isnan(loss_is) else got == loss_is).all()), (what, got)

    (ref, err), (rx, rx_err), _ = lce_ref(x[~hit], w, t[~hit], -100, torch.ones(int((~hit).sum()), device=DEV, dtype=torch.float64))
    plain = P.linear_cross_entropy(x, w, t, reduction="none")
    check(plain, "loss without gradients")
    within(plain[~hit], ref, err, "other rows' losses")
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = P.linear_cross_entropy(xs, ws, t, reduction="none")
    check(loss.detach(), "loss")
    within(loss.detach()[~hit], ref, err, "other rows' losses with gradients")
    dx, dw = torch.autograd.grad(loss, (xs, ws), torch.ones_like(loss))
    within(dx[~hit], rx, rx_err, "other rows' dx")
    if math.isnan(loss_is):
        assert torch.isnan(dx[hit]).all() and torch.isnan(dw).all()
    else:  # softmax - 1 with the target's share 0: z of the others as if it were not there
        W = w.double()
        z = (x.double() @ W.t())[hit]
        gone = z < -1e20
        assert bool(gone[:, v // 2].all())
        p = torch.softmax(z.masked_fill(gone, -math.inf), 1)
        p[:, v // 2] = -1.0
        zerr = ((24 + 64) * E * (x[hit, 2:].double().abs() @ W[:, 2:].abs().t())).amax(1, keepdim=True)
        rel = 4 * zerr + 2 * U[dtype] + (2 * v + 192) * E
        within(dx[hit], p @ W, rel * (p.abs() @ W.abs()) + U[dtype] * (p @ W).abs() + v * 2.0 ** -126 * W.abs().sum(0), "dx")
        assert torch.isfinite(dw[:, 2:]).all()
    for red in ("sum", "mean"):
        total = float(P.linear_cross_entropy(x, w, t, reduction=red))
        assert math.isnan(total) if math.isnan(loss_is) else total == math.inf


# -- launches of the largest calls --------------------------------------------------------------------------------------


def test_residual_norm_of_four_million_gates():
    """A gate for every two rows, so many that one workgroup for each would pass the 2^32 threads of a launch."""
    gates, d = 1 << 22, 8
    x, f, g = rnd((gates, 2, d), 1), rnd((gates, 2, d), 2), rnd((gates, 1, d), 3, std=0.5, mean=0.5)
    w = rnd(d, 4, std=0.1, mean=1.0)
    dy, dh = rnd((gates, 2, d), 5), rnd((gates, 2, d), 6)
    leaves = [q.requires_grad_() for q in (x, f, g, w)]
    y, h = P.residual_norm(x, f, gate=g, pre_weight=w, scale=0.5, eps=1e-5)
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))
    step = gates // 4
    for a in range(0, gates, step):  # (the reference in parts; the weight's gradient is the other tests')
        rows = [q.detach()[a:a + step].expand(step, 2, d).reshape(2 * step, d) for q in (x, f, g, dy, dh, y, h, grads[0], grads[1])]
        ref = res_ref(rows[0], rows[1], {"pre_weight": w.detach()}, "rms", None, rows[2], 0.5, 1e-5,
                      torch.ones_like(rows[0], dtype=torch.float64), rows[3], rows[4], U[torch.float32])
        for name, out in zip(("y", "h", "x", "f"), rows[5:]):
            within(out.detach(), *ref[name], name)
        dyt, dyt_err = ref["x"]  # the gate's gradient: the sum of scale dyt f over its two rows
        b = 0.5 * (dyt_err * rows[1].abs() + 10 * E * (dyt * rows[1]).abs()).view(step, 2, d).sum(1)
        v = 0.5 * (dyt * rows[1]).view(step, 2, d).sum(1)
        within(grads[2][a:a + step].view(step, d), v, b + U[torch.float32] * v.abs(), "gate")


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_entropy_of_sixteen_million_rows(dtype):
    """Two classes and so many rows that one workgroup for each would pass the 2^32 threads of a launch."""
    n, d, v = (1 << 24) + 5, 1, 2
    x, w, t = rnd((n, d), 1, dtype).requires_grad_(), rnd((v, d), 2, dtype).requires_grad_(), targets(n, v, 3, 0.1)
    loss = P.linear_cross_entropy(x, w, t, reduction="none")
    gx, gw = torch.autograd.grad(loss, (x, w), torch.ones_like(loss))
    (ref, err), (rx, rx_err), (rw, _) = lce_ref(x.detach(), w.detach(), t, -100, torch.ones(n, device=DEV, dtype=torch.float64))
    within(loss.detach(), ref, err, "loss")
    within(gx, rx, rx_err, "dx")
    # n roundings of partial sums, each within E of the terms' sum and either way: their sum grows with sqrt(n) (the bound
    # for roundings that all go one way would not see a lost part of the rows)
    terms = torch.stack([(p.abs() * x.detach().double().abs()[:, 0]).sum() for p in _dz(x.detach(), w.detach(), t)])[:, None]
    # (bf16: each logit's gradient is rounded, after its code's step of 2^-9, and so is the sum)
    within(gw, rw, (64 * math.sqrt(n) * E + (0 if dtype == torch.float32 else 3 * U[dtype])) * terms, "dw")


def _dz(x, w, t):
    """The logits' gradients of two classes in float64, a class at a time."""
    z = x.double() @ w.double().t()
    p = torch.softmax(z, 1)
    for c in (0, 1):
        yield torch.where(t == -100, 0.0, p[:, c] - (t == c).double())


# -- saved tensors ------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("way", ["checkpoint", "reentrant checkpoint", "on the host"])
def test_operators_under_checkpoints_and_saved_tensor_hooks(dtype, way):
    """The same bits where the forward pass is run again in the backward pass, and where saved tensors wait on the host."""
    x, f, w, t = rnd((600, 256), 1, dtype), rnd((600, 256), 2, dtype), rnd((1000, 256), 3, dtype, 0.1), targets(600, 1000, 4, 0.2)

    def loss(x, f, w):
        y, h = P.residual_norm(x, f, post="rms", p=0.1, seed=3)
        return P.linear_cross_entropy(P.dropout(h, 0.2, seed=4), w, t) / 3 + y.float().square().mean()

    def run(call):
        leaves = [q.detach().clone().requires_grad_() for q in (x, f, w)]
        out = call(*leaves)
        out.backward()
        return (out.detach(), *(q.grad for q in leaves))

    ref = run(loss)
    if way == "on the host":
        with torch.autograd.graph.save_on_cpu():
            out = run(loss)
    else:
        out = run(lambda *a: checkpoint(loss, *a, use_reentrant=way.startswith("reentrant")))
    assert all(torch.equal(p, q) for p, q in zip(ref, out))
