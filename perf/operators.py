"""The training operators of psgd_pro_amd as timed cases: linear_cross_entropy, residual_norm and dropout.

A case is a dict of plain values. kind "lce" is the loss of a language model's head (rows of x against a vocabulary matrix,
optionally with both gradients), "resnorm" the residual sum between two blocks of a transformer with its norms, gate, scale
and dropout, "drop" dropout by itself. `own` chooses between the package's operators and their plain forms in elementary
torch operations in float32; exact() computes the same outputs in float64 from the definitions.

Dropout: with a tensor seen as rows of its last dimension D, element (i, c) takes the 16-bit number c % 8 (low half of a word
first) of block i * ceil(D / 8) + c // 8 of Philox4x32-10 under the key (seed) and the upper counter words (stream); it is
kept where that number is at least round(65536 p) and then scaled by 65536 / (65536 - round(65536 p)).
"""
import math

import torch

own = False

DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
ESIZE = {"bf16": 2, "fp32": 4}
IGNORE = -100
EPS = 1e-6
M0, M1, W0, W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85
M32 = 0xFFFFFFFF


def _lce(name, n, d, v, dtype, grad, ignore):
    return dict(name=name, kind="lce", n=n, d=d, v=v, dtype=dtype, grad=grad, ignore=ignore)


def _res(name, batch, tokens, d, dtype, norm, post, gate, p, grad, scale=1.0):
    return dict(name=name, kind="resnorm", batch=batch, tokens=tokens, d=d, dtype=dtype, norm=norm, post=post, gate=gate,
                p=p, grad=grad, scale=scale)


def _drop(name, rows, d, dtype, p, grad):
    return dict(name=name, kind="drop", rows=rows, d=d, dtype=dtype, p=p, grad=grad)


def listed():
    return [
        # A micro-batch of a 4096-wide language model against a large vocabulary, some tokens padding: the largest call.
        _lce("lce_train_4096x4096x131072_bf16", 4096, 4096, 131072, "bf16", True, 0.1),
        # A narrow model with a medium vocabulary: the gradients' products are short or thin.
        _lce("lce_train_8192x768x32768_bf16", 8192, 768, 32768, "bf16", True, 0.0),
        # Nothing is a multiple of anything: packed sequences, an odd vocabulary, rows that are not 16-byte aligned, half of
        # the tokens (a prompt) not scored.
        _lce("lce_train_1531x770x50021_bf16", 1531, 770, 50021, "bf16", True, 0.5),
        # Full-precision training of a small model.
        _lce("lce_train_2048x512x10007_fp32", 2048, 512, 10007, "fp32", True, 0.0),
        # Evaluation: losses only.
        _lce("lce_score_2048x1024x65536_bf16", 2048, 1024, 65536, "bf16", False, 0.0),
        # The score of a single token: the vocabulary matrix is read once, nothing else counts.
        _lce("lce_score_1x4096x131072_bf16", 1, 4096, 131072, "bf16", False, 0.0),
        # Between two blocks of a 4096-wide model with norms on both sides of a block.
        _res("res_train_4x4096x4096_bf16", 4, 4096, 4096, "bf16", "rms", True, "none", 0.0, True),
        # The 512-wide vision transformer's residual in float32, with dropout and a learned scale for each channel.
        _res("res_train_512x65x512_fp32", 512, 65, 512, "fp32", "layer", False, "channel", 0.1, True),
        # Gates of each sequence on 770 channels: no row is a multiple of a vector.
        _res("res_train_33x257x770_bf16", 33, 257, 770, "bf16", "layer", True, "sequence", 0.0, True, 0.5),
        # One token of a generation step: a call's fixed cost.
        _res("res_token_1x1x4096_bf16", 1, 1, 4096, "bf16", "rms", True, "none", 0.0, False),
        # Dropout on the activations of a large batch.
        _drop("drop_train_16384x4096_bf16", 16384, 4096, "bf16", 0.1, True),
        # Dropout on a small ragged batch.
        _drop("drop_train_333x770_fp32", 333, 770, "fp32", 0.25, True),
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm of lo..hi, every second one a multiple of 64 where that is in range."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 64:
        v = v // 64 * 64
    return min(hi, max(lo, v))


def draw(rng):
    kind = rng.choice(["lce", "lce", "resnorm", "resnorm", "drop"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    if kind == "lce":
        n, d, v = _size(rng, 1, 8192), _size(rng, 256, 4096), _size(rng, 1000, 131072)
        while n * d * v > 2 ** 40 or (dtype == "fp32" and n * d * v > 2 ** 37):
            n = max(1, n // 2)
        return dict(kind="lce", n=n, d=d, v=v, dtype=dtype, grad=rng.random() < 0.6, ignore=rng.choice([0.0, 0.1, 0.5]))
    if kind == "resnorm":
        batch, tokens, d = _size(rng, 1, 64), _size(rng, 1, 4096), _size(rng, 256, 8192)
        while batch * tokens * d > 2 ** 26:
            tokens = max(1, tokens // 2)
        return dict(kind="resnorm", batch=batch, tokens=tokens, d=d, dtype=dtype, norm=rng.choice(["rms", "layer"]),
                    post=rng.random() < 0.5, gate=rng.choice(["none", "channel", "sequence", "token"]),
                    p=rng.choice([0.0, 0.0, 0.1]), grad=rng.random() < 0.7, scale=rng.choice([1.0, 0.5]))
    rows, d = _size(rng, 1, 16384), _size(rng, 256, 4096)
    return dict(kind="drop", rows=rows, d=d, dtype=dtype, p=rng.choice([0.05, 0.1, 0.25, 0.5]), grad=rng.random() < 0.7)


def _gate_shape(case):
    b, t, d = case["batch"], case["tokens"], case["d"]
    return {"none": None, "channel": (d,), "sequence": (b, 1, d), "token": (b, t, d)}[case["gate"]]


def prepare(case, seed):
    """Inputs as a training step has them: normalised rows against a vocabulary matrix of standard deviation 0.02 d^(-1/2)
    sqrt(4096), half of the rows pulled towards their target as a trained model's are; unit-variance activations with a
    few large channels, weights near 1, gates near 0.5."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DT[case["dtype"]]
    leaf = case["grad"]

    def rnd(*shape, std=1.0, mean=0.0, dtype=dt, grad=leaf):
        t = torch.randn(shape, generator=g, device=DEV).mul_(std).add_(mean).to(dtype)
        return t.requires_grad_(grad)

    st = dict(case=case, drop_seed=seed * 7919 + 12345, stream=seed % 5)
    if case["kind"] == "lce":
        n, d, v = case["n"], case["d"], case["v"]
        w = rnd(v, d, std=1.28 / math.sqrt(d), grad=False)
        t = torch.randint(v, (n,), generator=g, device=DEV)
        pull = torch.rand((n, 1), generator=g, device=DEV).mul_(24).sub_(12).clamp_(min=0) / 1.28 ** 2
        x = (torch.randn((n, d), generator=g, device=DEV) + pull * w[t].float()).to(dt)
        skip = torch.rand((n,), generator=g, device=DEV) < case["ignore"]
        st.update(x=x.requires_grad_(leaf), w=w.requires_grad_(leaf), t=t.masked_fill(skip, IGNORE))
    elif case["kind"] == "resnorm":
        b, t, d = case["batch"], case["tokens"], case["d"]
        big = 1 + 9 * (torch.rand((d,), generator=g, device=DEV) < 0.01).float()
        st["x"] = (torch.randn((b, t, d), generator=g, device=DEV) * big).to(dt).requires_grad_(leaf)
        st["f"] = rnd(b, t, d, std=0.5, mean=0.05)
        names = ["pre_weight"] + ["post_weight"] * case["post"]
        if case["norm"] == "layer":
            names += ["pre_bias"] + ["post_bias"] * case["post"]
        st["par"] = {k: rnd(d, std=0.1, mean=1.0 if k.endswith("weight") else 0.0, dtype=torch.float32) for k in names}
        if case["gate"] != "none":
            st["par"]["gate"] = rnd(*_gate_shape(case), std=0.25, mean=0.5)
        st["dy"], st["dh"] = rnd(b, t, d, grad=False), rnd(b, t, d, grad=False)
    else:
        st["x"] = rnd(case["rows"], case["d"])
        st["dy"] = rnd(case["rows"], case["d"], grad=False)
    return st


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------


def _mask_scale(rows, d, p, seed, stream, dev):
    """rows x d factors: 0 where dropped, else the scale. 64-bit integer products wrap; their low 64 bits are exact."""
    nb = (d + 7) // 8
    thr = round(65536 * p)
    blk = torch.arange(rows * nb, device=dev)
    c0, c1 = blk & M32, blk >> 32
    c2, c3 = torch.full_like(blk, stream & M32), torch.full_like(blk, (stream >> 32) & M32)
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(10):
        p0, p1 = c0 * M0, c2 * M1
        c0, c1, c2, c3 = ((p1 >> 32) & M32) ^ c1 ^ k0, p1 & M32, ((p0 >> 32) & M32) ^ c3 ^ k1, p0 & M32
        k0, k1 = (k0 + W0) & M32, (k1 + W1) & M32
    words = torch.stack((c0 & 65535, c0 >> 16, c1 & 65535, c1 >> 16, c2 & 65535, c2 >> 16, c3 & 65535, c3 >> 16), 1)
    keep = (words >= thr).view(rows, nb * 8)[:, :d]
    return keep.float() * (65536.0 / (65536 - thr))


def _plain_lce(st):
    case = st["case"]
    with torch.no_grad():
        x, w, t = st["x"].float(), st["w"].float(), st["t"]
        valid = t != IGNORE
        rows = torch.arange(t.numel(), device=t.device)
        tt = torch.where(valid, t, 0)
        inv = 1.0 / valid.sum().clamp(min=1)
        z = x @ w.t()
        mx = z.max(1).values
        zt = z[rows, tt]
        e = z.sub_(mx[:, None]).exp_()
        s = e.sum(1)
        each = torch.where(valid, s.log() + mx - zt, 0.0)
        if not case["grad"]:
            return each
        e *= (torch.where(valid, inv, 0.0) / s)[:, None]
        e[rows, tt] -= torch.where(valid, inv, 0.0)
        return each.sum() * inv, (e @ w).to(st["x"].dtype), (e.t() @ x).to(st["w"].dtype)


def _plain_norm(v, kind, weight, bias):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * (v.square().mean(-1, keepdim=True) + EPS).rsqrt() * weight
    return v if bias is None else v + bias


def _plain_res(st):
    case, par = st["case"], st["par"]
    x, b = st["x"].float(), st["f"].float()
    if case["post"]:
        b = _plain_norm(b, case["norm"], par["post_weight"], par.get("post_bias"))
    if case["p"] > 0:
        m = _mask_scale(case["batch"] * case["tokens"], case["d"], case["p"], st["drop_seed"], st["stream"], x.device)
        b = b * m.view(b.shape)
    if case["gate"] != "none":
        b = b * par["gate"].float()
    y = x + case["scale"] * b
    h = _plain_norm(y, case["norm"], par["pre_weight"], par.get("pre_bias"))
    return y.to(st["x"].dtype), h.to(st["x"].dtype)


def _plain_drop(st):
    case = st["case"]
    m = _mask_scale(case["rows"], case["d"], case["p"], st["drop_seed"], st["stream"], st["x"].device)
    return (st["x"].float() * m).to(st["x"].dtype)


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------


def _own_forward(st):
    import psgd_pro_amd as P
    case = st["case"]
    if case["kind"] == "lce":
        return P.linear_cross_entropy(st["x"], st["w"], st["t"], ignore_index=IGNORE,
                                      reduction="mean" if case["grad"] else "none")
    if case["kind"] == "resnorm":
        return P.residual_norm(st["x"], st["f"], pre=case["norm"], post=case["norm"] if case["post"] else None,
                               scale=case["scale"], eps=EPS, p=case["p"], seed=st["drop_seed"], stream=st["stream"],
                               **st["par"])
    return P.dropout(st["x"], case["p"], seed=st["drop_seed"], stream=st["stream"])


def run(state):
    case = state["case"]
    if not own and case["kind"] == "lce":
        return _plain_lce(state)
    forward = _own_forward if own else (_plain_res if case["kind"] == "resnorm" else _plain_drop)
    if not case["grad"]:
        with torch.no_grad():
            return forward(state)
    out = forward(state)
    if case["kind"] == "lce":
        return (out.detach(), *torch.autograd.grad(out, (state["x"], state["w"])))
    if case["kind"] == "drop":
        return (out.detach(), *torch.autograd.grad(out, state["x"], state["dy"]))
    y, h = out
    leaves = (state["x"], state["f"], *state["par"].values())
    return (y.detach(), h.detach(), *torch.autograd.grad((y, h), leaves, (state["dy"], state["dh"])))


def work(case):
    e = ESIZE[case["dtype"]]
    if case["kind"] == "lce":
        n, d, v = case["n"], case["d"], case["v"]
        return {"bytes": (n + v) * d * e * (2 if case["grad"] else 1) + 12 * n, "flops": (6 if case["grad"] else 2) * n * d * v}
    if case["kind"] == "drop":
        x = case["rows"] * case["d"]
        return {"bytes": (4 if case["grad"] else 2) * x * e, "flops": (2 if case["grad"] else 1) * x}
    x = case["batch"] * case["tokens"] * case["d"]
    gate = {"none": 0, "channel": case["d"], "sequence": case["batch"] * case["d"], "token": x}[case["gate"]]
    par = case["d"] * 4 * (1 + case["post"]) * (2 if case["norm"] == "layer" else 1)
    # forward: x, f in, y, h out; backward: dy, dh in, dx, df out (x, f and what the forward made are counted once)
    return {"bytes": (8 if case["grad"] else 4) * x * e + (gate * e + par) * (2 if case["grad"] else 1),
            "flops": (40 if case["grad"] else 12) * x}


# ---------------------------------------------------------------------------------------------------------------------
# float64
# ---------------------------------------------------------------------------------------------------------------------


def _factors64(case, st, rows, d):
    """The dropout factors again, the 32 x 32-bit products by 16-bit halves, one number of each block at a time."""
    per_row = -(-d // 8)
    i = torch.arange(rows, device=DEV).repeat_interleave(per_row) * per_row + torch.arange(per_row, device=DEV).repeat(rows)
    ctr = [i % 2 ** 32, i // 2 ** 32, torch.zeros_like(i) + st["stream"] % 2 ** 32, torch.zeros_like(i) + st["stream"] // 2 ** 32]
    key = [st["drop_seed"] % 2 ** 32, st["drop_seed"] // 2 ** 32 % 2 ** 32]

    def high_low(a, m):
        mh, ml = m // 65536, m % 65536
        ah, al = a // 65536, a % 65536
        low = al * ml
        mid = ah * ml + low // 65536
        mid2 = al * mh + mid % 65536
        return ah * mh + mid // 65536 + mid2 // 65536, mid2 % 65536 * 65536 + low % 65536

    for r in range(10):
        h0, l0 = high_low(ctr[0], M0)
        h1, l1 = high_low(ctr[2], M1)
        ctr = [h1 ^ ctr[1] ^ key[0], l1, h0 ^ ctr[3] ^ key[1], l0]
        key = [(key[0] + W0) % 2 ** 32, (key[1] + W1) % 2 ** 32]
    lost = int(math.floor(65536 * case["p"] + 0.5))
    out = torch.empty(rows * per_row, 8, device=DEV, dtype=torch.float64)
    for c in range(8):
        out[:, c] = (ctr[c // 2] // (65536 if c % 2 else 1) % 65536 >= lost).double() * (65536 / (65536 - lost))
    return out.reshape(rows, per_row * 8)[:, :d]


def _exact_lce(case, st):
    x, w, t = st["x"].detach().double(), st["w"].detach().double(), st["t"]
    count = max(1, int((t != IGNORE).sum()))
    each = torch.zeros(case["n"], device=DEV, dtype=torch.float64)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for a in range(0, case["n"], 1024):
        rows = torch.nonzero(t[a:a + 1024] != IGNORE).flatten() + a
        if not rows.numel():
            continue
        z = x[rows] @ w.t()
        own_z = z.gather(1, t[rows, None])
        lse = torch.logsumexp(z, 1, keepdim=True)
        each[rows] = (lse - own_z).flatten()
        if case["grad"]:
            dz = torch.exp(z - lse) / count
            # softmax - 1 at the target, from the sum of the others
            others = torch.exp(z - lse).scatter_(1, t[rows, None], 0.0).sum(1, keepdim=True)
            dz.scatter_(1, t[rows, None], -others / count)
            dx[rows] = dz @ w
            dw += dz.t() @ x[rows]
    return (each.sum() / count, dx, dw) if case["grad"] else each


def _norm64(v, kind, weight, bias):
    """The norm and what its derivative needs."""
    c = v - v.mean(1, keepdim=True) if kind == "layer" else v
    rstd = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    hat = c * rstd
    return hat * weight + (0 if bias is None else bias), hat, rstd


def _norm_grad64(g, kind, weight, hat, rstd):
    c = g * weight
    out = c - hat * (c * hat).mean(1, keepdim=True)
    if kind == "layer":
        out = out - c.mean(1, keepdim=True)
    return out * rstd, (g * hat).sum(0), g.sum(0)


def _exact_res(case, st):
    rows, d, kind = case["batch"] * case["tokens"], case["d"], case["norm"]
    flat = {k: st[k].detach().double().reshape(rows, d) for k in ("x", "f", "dy", "dh")}
    par = {k: v.detach().double() for k, v in st["par"].items()}
    shape = st["x"].shape
    u, b = None, flat["f"]
    if case["post"]:
        b, u, u_rstd = _norm64(b, kind, par["post_weight"], par.get("post_bias"))
    keep = _factors64(case, st, rows, d) if case["p"] > 0 else 1.0
    b = b * keep
    gate = par["gate"].expand(shape).reshape(rows, d) if "gate" in par else 1.0
    y = flat["x"] + case["scale"] * gate * b
    h, hat, rstd = _norm64(y, kind, par["pre_weight"], par.get("pre_bias"))
    if not case["grad"]:
        return y.view(shape), h.view(shape)
    through, d_pre_w, d_pre_b = _norm_grad64(flat["dh"], kind, par["pre_weight"], hat, rstd)
    dx = flat["dy"] + through
    df = case["scale"] * gate * keep * dx
    grads = {"pre_weight": d_pre_w, "pre_bias": d_pre_b}
    if "gate" in par:
        grads["gate"] = (case["scale"] * dx * b).view(shape).sum_to_size(par["gate"].shape)
    if case["post"]:
        df, grads["post_weight"], grads["post_bias"] = _norm_grad64(df, kind, par["post_weight"], u, u_rstd)
    return (y.view(shape), h.view(shape), dx.view(shape), df.view(shape), *(grads[k] for k in st["par"]))


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "lce":
            return _exact_lce(case, st)
        if case["kind"] == "resnorm":
            return _exact_res(case, st)
        m = _factors64(case, st, case["rows"], case["d"])
        y = st["x"].detach().double() * m
        return (y, st["dy"].double() * m) if case["grad"] else y
