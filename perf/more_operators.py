"""More operators of psgd_pro_amd as timed cases: window_attention, qk_norm_rope and adamw_step.

A case is a dict of plain values. kind "attn" is attention with a sliding window and first tokens that stay visible (training
with its gradients, or single tokens over a cache), "rope" the norms of queries and keys for each head with the position
rotation, "adamw" one step over all tensors of a model with its states in 32 or 8 bits. `own` chooses between the package's
operators and their plain forms in elementary torch operations in float32; exact() computes the same outputs in float64 from
the definitions.

attn: the query at position p of a sequence of `length` tokens sees key j where j <= p, j < length, p < length and
(p - j < window or j < sinks); a query that sees none has output 0. Head h takes the keys of head h // (heads / kv_heads).

adamw with 8 bits: a state is held in e4m3 codes with one power-of-two scale for each 256 elements of a tensor, the first
moment m as it is and the second as its root. With E the exponent field of the largest magnitude of the block (one more where
its mantissa is over 1.75) the scale's exponent field is max(E - 8, 1), and 0 where the block is zero. A magnitude is rounded
to the code below or above by a 16-bit number: its bits below the code's lowest, plus 16 times that number, carry or not.
Element i of tensor t at step s takes the number i % 8 (low half of a word first) of block i // 8 of Philox4x32-10 under the
key (seed) and the upper counter words (s, t). A root that is not 0 has no code 0.
"""
import math

import torch

own = False

DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
ESIZE = {"bf16": 2, "fp32": 4}
EPS = 1e-6
LR, BETA1, BETA2, ADAM_EPS, DECAY, STEP = 1e-3, 0.9, 0.999, 1e-8, 0.1, 10
M0, M1, W0, W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85
M32 = 0xFFFFFFFF
BLOCK = 256


def _attn(name, batch, queries, keys, heads, kv, d, dtype, window, sinks, ragged, grad):
    return dict(name=name, kind="attn", batch=batch, queries=queries, keys=keys, heads=heads, kv=kv, d=d, dtype=dtype,
                window=window, sinks=sinks, ragged=ragged, grad=grad)


def _rope(name, batch, tokens, heads, kv, d, rot, dtype, norm, interleaved, far, grad):
    return dict(name=name, kind="rope", batch=batch, tokens=tokens, heads=heads, kv=kv, d=d, rot=rot, dtype=dtype, norm=norm,
                interleaved=interleaved, far=far, grad=grad)


def _adamw(name, layers, d, ff, vocab, dtype, bits, clip):
    return dict(name=name, kind="adamw", layers=layers, d=d, ff=ff, vocab=vocab, dtype=dtype, bits=bits, clip=clip)


def listed():
    return [
        # A micro-batch of a 4096-wide language model with grouped heads, all earlier tokens visible: the largest call.
        _attn("attn_train_4x4096_32over8x128_bf16", 4, 4096, 4096, 32, 8, 128, "bf16", 0, 0, False, True),
        # A long text under a window of 1024 with four first tokens kept: few keys a query, but four keys with all queries.
        _attn("attn_train_1x16384_16over4x64_w1024_bf16", 1, 16384, 16384, 16, 4, 64, "bf16", 1024, 4, False, True),
        # Full-precision training of a small model on a padded batch: odd lengths, odd heads, heads of 80.
        _attn("attn_train_3x1021_9over3x80_w300_fp32", 3, 1021, 1021, 9, 3, 80, "fp32", 300, 2, True, True),
        # A generation step of 32 sequences of different lengths over their caches.
        _attn("attn_token_32x1over8192_32over8x128_w4096_bf16", 32, 1, 8192, 32, 8, 128, "bf16", 4096, 4, True, False),
        # One token of one sequence over a long cache: the keys are read once, nothing else counts.
        _attn("attn_token_1x1over131072_32over8x128_bf16", 1, 1, 131072, 32, 8, 128, "bf16", 0, 0, False, False),
        # The same model's queries and keys, between its projection and its attention.
        _rope("rope_train_4x4096_32over8x128_bf16", 4, 4096, 32, 8, 128, 128, "bf16", "rms", False, 0, True),
        # Nothing is a power of two, half of a head is rotated, pairs side by side, layer norms.
        _rope("rope_train_3x1021_9over3x80_fp32", 3, 1021, 9, 3, 80, 40, "fp32", "layer", True, 0, True),
        # The generation step's tokens, far into their texts: a call's fixed cost.
        _rope("rope_token_32x1_32over8x128_bf16", 32, 1, 32, 8, 128, 128, "bf16", "rms", False, 1 << 20, False),
        # The step of a half-billion-parameter model in float32, its gradients clipped.
        _adamw("adamw_8x2048_fp32", 8, 2048, 5632, 32768, "fp32", 32, True),
        # The same model in bfloat16 with states of 8 bits: a third of the bytes.
        _adamw("adamw_8x2048_bf16_8bit", 8, 2048, 5632, 32768, "bf16", 8, False),
        # Odd widths, tensors packed one after the other on no boundary, 8 bits.
        _adamw("adamw_2x770_fp32_8bit", 2, 770, 1531, 5003, "fp32", 8, False),
        # What a Kron preconditioner does not take of a 512-wide model, norms and gates: many short tensors.
        _adamw("adamw_vectors_48x512_fp32", 48, 512, 0, 0, "fp32", 32, True),
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm of lo..hi, every second one a multiple of 64 where that is in range."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v >= 64:
        v = v // 64 * 64
    return min(hi, max(lo, v))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "rope", "rope", "adamw", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    kv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4, 5])
    heads, d = kv * group, rng.choice([32, 64, 64, 72, 80, 96, 128, 128])
    if kind == "attn":
        window = rng.choice([0, 0, _size(rng, 16, 4096)])
        sinks = rng.choice([0, 1, 4, 77])
        if rng.random() < 0.6:
            batch, n = _size(rng, 1, 8), _size(rng, 1, 8192)
            while batch * heads * n * n > 2 ** 31 or (dtype == "fp32" and batch * heads * n * n > 2 ** 28):
                n = max(1, n * 3 // 4)
            return dict(kind="attn", batch=batch, queries=n, keys=n, heads=heads, kv=kv, d=d, dtype=dtype, window=window,
                        sinks=sinks, ragged=rng.random() < 0.5, grad=rng.random() < 0.7)
        batch, queries, keys = _size(rng, 1, 64), rng.choice([1, 1, 1, 2, 7]), _size(rng, 8, 131072)
        while batch * keys * kv > 2 ** 21:
            keys = max(8, keys // 2)
        return dict(kind="attn", batch=batch, queries=queries, keys=keys, heads=heads, kv=kv, d=d, dtype=dtype, window=window,
                    sinks=sinks, ragged=rng.random() < 0.5, grad=False)
    if kind == "rope":
        batch, tokens = _size(rng, 1, 64), _size(rng, 1, 8192)
        while batch * tokens * (heads + kv) * d > 2 ** 26:
            tokens = max(1, tokens // 2)
        return dict(kind="rope", batch=batch, tokens=tokens, heads=heads, kv=kv, d=d, rot=rng.choice([d, d, d // 2]), dtype=dtype,
                    norm=rng.choice(["rms", "rms", "layer"]), interleaved=rng.random() < 0.3, far=rng.choice([0, 0, 1 << 20]),
                    grad=rng.random() < 0.6)
    bits = rng.choice([8, 32])
    layers, d, ff, vocab = _size(rng, 1, 24), _size(rng, 64, 2048), rng.choice([0, _size(rng, 64, 5632)]), _size(rng, 100, 32768)
    while layers * d * (4 * d + 2 * ff) * (ff > 0) + vocab * d > 2 ** 28:
        layers, vocab = max(1, layers // 2), max(100, vocab // 2)
    return dict(kind="adamw", layers=layers, d=d, ff=ff, vocab=rng.choice([0, vocab]) if ff else 0, dtype=dtype, bits=bits,
                clip=bits == 32 and rng.random() < 0.5)


def _shapes(case):
    """The tensors of a model: embeddings, of each layer four matrices (ff 0: none), two norms and two gates; a last norm."""
    d, ff = case["d"], case["ff"]
    layer = [(3 * d, d), (d, d), (ff, d), (d, ff)] * (ff > 0) + [(d,)] * 4
    return [(case["vocab"], d)] * (case["vocab"] > 0) + layer * case["layers"] + [(d,)]


def _views(flat, shapes):
    """Tensors of these shapes one after the other in `flat`."""
    return [t.view(s) for t, s in zip(flat[:sum(math.prod(s) for s in shapes)].split([math.prod(s) for s in shapes]), shapes)]


def prepare(case, seed):
    """Inputs as a model has them: queries, keys and values as the parts of one projection (or keys and values in caches with
    room behind the last token), heads of unit variance with a few large channels before their norms, weights near 1; gradients
    of sizes that differ by tensor and are heavy-tailed, states as after some steps of the same gradients."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    st = dict(case=case)
    if case["kind"] == "adamw":
        shapes = _shapes(case)
        n = sum(math.prod(s) for s in shapes)
        dt = DT[case["dtype"]]
        size = torch.exp(torch.randn(len(shapes), generator=g, device=DEV)).mul_(1e-3)
        size = size.repeat_interleave(torch.tensor([math.prod(s) for s in shapes], device=DEV), output_size=n)
        p = torch.randn(n, generator=g, device=DEV).mul_(0.05).to(dt)
        grad = torch.randn(n, generator=g, device=DEV).mul_(size)
        old = torch.randn(n, generator=g, device=DEV)
        root = size.mul_(torch.rand(n, generator=g, device=DEV).add_(0.5))
        st.update(shapes=shapes, seed=seed * 7919 + 12345, p=p, g=grad.to(dt), params=_views(p, shapes))
        st["grads"] = _views(st["g"], shapes)
        if case["bits"] == 32:
            st["m"], st["v"] = old.mul_(root).mul_(0.3), root.square_()
            st["ms"], st["vs"] = _views(st["m"], shapes), _views(st["v"], shapes)
            return st
        # codes within one block's scale: a magnitude below 448 for roots, both signs for the first moment
        blocks = [-(-math.prod(s) // BLOCK) for s in shapes]
        st["m"] = old.mul_(60).clamp_(-448, 448).to(torch.float8_e4m3fn)
        st["v"] = root.mul_(3e4).clamp_(2 ** -9, 448).to(torch.float8_e4m3fn)
        st["m_scale"] = torch.full((sum(blocks),), 105, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
        st["v_scale"] = torch.full((sum(blocks),), 111, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
        flat = [(math.prod(s),) for s in shapes]
        part = [(b,) for b in blocks]
        st["ms"] = list(zip(_views(st["m"], flat), _views(st["m_scale"], part)))
        st["vs"] = list(zip(_views(st["v"], flat), _views(st["v_scale"], part)))
        return st
    dt, leaf = DT[case["dtype"]], case["grad"]
    b, h, kv, d = case["batch"], case["heads"], case["kv"], case["d"]

    def rnd(*shape, std=1.0, mean=0.0, dtype=dt):
        return torch.randn(shape, generator=g, device=DEV).mul_(std).add_(mean).to(dtype)

    if case["kind"] == "rope":
        n = case["tokens"]
        x = torch.randn((b, n, h + 2 * kv, d), generator=g, device=DEV)
        x = x.mul_(1 + 9 * (torch.rand((d,), generator=g, device=DEV) < 0.02).float()).add_(0.05).to(dt)
        st["q"], st["k"] = x[:, :, :h].requires_grad_(leaf), x[:, :, h:h + kv].requires_grad_(leaf)
        st["qw"], st["kw"] = (rnd(d, std=0.1, mean=1.0, dtype=torch.float32).requires_grad_(leaf) for _ in range(2))
        st["dq"], st["dk"] = rnd(b, n, h, d), rnd(b, n, kv, d)
        start = torch.randint(case["far"] + 1, (b, 1), generator=g, device=DEV)
        st["pos"] = start + torch.arange(n, device=DEV)
        return st
    n, m = case["queries"], case["keys"]
    if n == m:
        x = torch.randn((b, n, h + 2 * kv, d), generator=g, device=DEV).to(dt)
        st["q"], st["k"], st["v"] = (t.requires_grad_(leaf) for t in x.split((h, kv, kv), 2))
    else:
        st["q"], st["k"], st["v"] = rnd(b, n, h, d), rnd(b, m, kv, d), rnd(b, m, kv, d)
    st["do"] = rnd(b, n, h, d)
    st["lengths"] = st["starts"] = None
    if case["ragged"]:
        st["lengths"] = torch.randint(min(n, max(1, m // 2)), m + 1, (b,), generator=g, device=DEV)
        st["starts"] = None if n == m else st["lengths"] - n
    return st


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------


def _visible(st):
    """(batch, queries, keys): what each query sees."""
    case, m = st["case"], st["case"]["keys"]
    i, j = torch.arange(case["queries"], device=DEV), torch.arange(m, device=DEV)
    lengths = torch.full((case["batch"],), m, device=DEV) if st["lengths"] is None else st["lengths"]
    starts = torch.full((case["batch"],), m - case["queries"], device=DEV) if st["starts"] is None else st["starts"]
    pos = (starts[:, None] + i)[:, :, None]
    length = lengths[:, None, None]
    seen = (j <= pos) & (j < length) & (pos < length)
    return seen & ((pos - j < case["window"]) | (j < case["sinks"])) if case["window"] else seen


def _plain_attn(st):
    case, dt = st["case"], st["q"].dtype
    b, n, m, kv, d = case["batch"], case["queries"], case["keys"], case["kv"], case["d"]
    group = case["heads"] // kv
    with torch.no_grad():
        def rows(t):  # (batch, kv heads, group * tokens, d)
            return t.float().view(b, t.shape[1], kv, -1, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d)

        def back(t, tokens):
            return t.view(b, kv, -1, tokens, d).permute(0, 3, 1, 2, 4).reshape(b, tokens, -1, d).to(dt)

        q, k, v = rows(st["q"]), rows(st["k"]), rows(st["v"])
        scale = 1 / math.sqrt(d)
        s = (q @ k.transpose(2, 3)).mul_(scale).view(b, kv, group, n, m)
        s.masked_fill_(~_visible(st)[:, None, None], -math.inf)
        top = s.amax(-1, keepdim=True)
        p = s.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
        total = p.sum(-1, keepdim=True)
        p = p.div_(total.masked_fill_(total == 0, 1.0)).view(b, kv, group * n, m)
        o = p @ v
        if not case["grad"]:
            return back(o, n)
        do = rows(st["do"])
        dv = p.transpose(2, 3) @ do
        ds = (do @ v.transpose(2, 3)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
        return back(o, n), back(ds @ k * scale, n), back(ds.transpose(2, 3) @ q * scale, m), back(dv, m)


def _rotate(t, case, pos):
    rot = case["rot"]
    turn = pos.double()[:, :, None, None] * 10000.0 ** (torch.arange(0, rot, 2, device=DEV).double() / -rot)
    cos, sin = turn.cos().float(), turn.sin().float()
    if case["interleaved"]:
        a, c = t[..., 0:rot:2], t[..., 1:rot:2]
        r = torch.stack((a * cos - c * sin, c * cos + a * sin), -1).flatten(-2)
    else:
        a, c = t[..., :rot // 2], t[..., rot // 2:rot]
        r = torch.cat((a * cos - c * sin, c * cos + a * sin), -1)
    return torch.cat((r, t[..., rot:]), -1)


def _plain_rope(st):
    case = st["case"]

    def one(x, w):
        v = x.float()
        if case["norm"] == "layer":
            v = v - v.mean(-1, keepdim=True)
        return _rotate(v * (v.square().mean(-1, keepdim=True) + EPS).rsqrt() * w, case, st["pos"]).to(x.dtype)

    return one(st["q"], st["qw"]), one(st["k"], st["kw"])


def _numbers(n, seed, step, tensor):
    """One 16-bit number for each of n elements. 64-bit integer products wrap; their low 64 bits are exact."""
    c0 = torch.arange((n + 7) // 8, device=DEV)
    c1, c2, c3 = torch.zeros_like(c0), torch.full_like(c0, step), torch.full_like(c0, tensor)
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(10):
        p0, p1 = c0 * M0, c2 * M1
        c0, c1, c2, c3 = ((p1 >> 32) & M32) ^ c1 ^ k0, p1 & M32, ((p0 >> 32) & M32) ^ c3 ^ k1, p0 & M32
        k0, k1 = (k0 + W0) & M32, (k1 + W1) & M32
    words = torch.stack((c0 & 65535, c0 >> 16, c1 & 65535, c1 >> 16, c2 & 65535, c2 >> 16, c3 & 65535, c3 >> 16), 1)
    return words.int().view(-1)[:n]


def _unpack(codes, scales):
    return codes.float() * scales.float().repeat_interleave(BLOCK)[:codes.numel()]


def _pack(x, numbers, root, codes, scales):
    """x (float32) into codes and scales, as the module's text says."""
    blocks = scales.numel()
    padded = torch.zeros(blocks * BLOCK, device=DEV)
    padded[:x.numel()] = x.abs()
    top = padded.view(blocks, BLOCK).amax(1)
    field = torch.where(top > 0, ((top.view(torch.int32) + 0x1FFFFF) >> 23).sub(8).clamp(min=1), 0)
    scales.view(torch.uint8).copy_(field)
    up = ((254 - field) << 23).view(torch.float32).repeat_interleave(BLOCK)[:x.numel()]
    mag = ((x.abs() * up * 2.0 ** -120).view(torch.int32) + numbers * 16) >> 20
    if root:
        mag = torch.maximum(mag, (x > 0).int())
    codes.view(torch.uint8).copy_(torch.where(x < 0, mag + 128, mag))


def _plain_adamw(st):
    case = st["case"]
    c1, c2 = 1 - BETA1 ** STEP, 1 - BETA2 ** STEP

    def step(p, g, m, v):
        m = m * BETA1 + g * (1 - BETA1)
        v = v * BETA2 + g * g * (1 - BETA2)
        p.copy_(p.float() * (1 - LR * DECAY) - LR * (m / c1) / ((v / c2).sqrt() + ADAM_EPS))
        return m, v

    if case["bits"] == 32:
        g = st["g"].float()
        norm = g.double().square().sum().sqrt() if case["clip"] else None
        if case["clip"]:
            g = g * (1.0 / norm).clamp(max=1.0).float()
        m, v = step(st["p"], g, st["m"], st["v"])
        st["m"].copy_(m)
        st["v"].copy_(v)
        return (st["p"], st["m"], st["v"]) + ((norm.float(),) if case["clip"] else ())
    for i, (p, g, m, v) in enumerate(zip(st["params"], st["grads"], st["ms"], st["vs"])):
        mean, var = step(p.view(-1), g.reshape(-1).float(), _unpack(*m), _unpack(*v).square())
        numbers = _numbers(p.numel(), st["seed"], STEP, i)
        _pack(mean, numbers, False, *m)
        _pack(var.double().sqrt().float(), numbers, True, *v)
    return st["p"], st["m"], st["m_scale"], st["v"], st["v_scale"]


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------


def _own_forward(st):
    import psgd_pro_amd as P
    case = st["case"]
    if case["kind"] == "attn":
        return P.window_attention(st["q"], st["k"], st["v"], window=case["window"] or None, sinks=case["sinks"],
                                  lengths=st["lengths"], starts=st["starts"])
    if case["kind"] == "rope":
        return P.qk_norm_rope(st["q"], st["k"], norm=case["norm"], q_weight=st["qw"], k_weight=st["kw"], eps=EPS,
                              positions=st["pos"], theta=10000.0, rotary_dim=case["rot"], interleaved=case["interleaved"])
    norm = P.adamw_step(st["params"], st["grads"], st["ms"], st["vs"], step=STEP, lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS,
                        weight_decay=DECAY, max_norm=1.0 if case["clip"] else None, seed=st.get("seed", 0))
    if case["bits"] == 8:
        return st["p"], st["m"], st["m_scale"], st["v"], st["v_scale"]
    return (st["p"], st["m"], st["v"]) + ((norm,) if case["clip"] else ())


def run(state):
    case = state["case"]
    if not own and case["kind"] == "attn":
        return _plain_attn(state)
    forward = _own_forward if own else (_plain_rope if case["kind"] == "rope" else _plain_adamw)
    if not case.get("grad"):
        with torch.no_grad():
            return forward(state)
    out = forward(state)
    if case["kind"] == "attn":
        return (out.detach(), *torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["do"]))
    q, k = out
    leaves = (state["q"], state["k"], state["qw"], state["kw"])
    return (q.detach(), k.detach(), *torch.autograd.grad((q, k), leaves, (state["dq"], state["dk"])))


def _pairs(case):
    """Keys that the queries of one head see, over the batch (sequences of different lengths: as if all were three quarters
    of the longest)."""
    n, m, w, s = case["queries"], case["keys"], case["window"], case["sinks"]
    m = m * 3 // 4 if case["ragged"] else m
    n = min(n, m)
    total = 0
    for p in range(m - n, m):
        seen = min(p + 1, w) if w else p + 1
        total += seen + (min(s, p + 1 - seen) if w else 0)
    return case["batch"] * total


def work(case):
    e = ESIZE[case["dtype"]]
    if case["kind"] == "attn":
        n, h, kv, d = case["batch"] * case["queries"], case["heads"], case["kv"], case["d"]
        pairs = _pairs(case)
        keys = case["batch"] * case["keys"] * kv if n > case["batch"] * 64 else min(pairs, case["batch"] * case["keys"]) * kv
        q, k = n * h * d * e, keys * d * e
        # forward: q, k, v in, o out; backward: do in, dq, dk, dv out (q, k, v, o are counted once)
        return {"bytes": (4 if case["grad"] else 2) * (q + k), "flops": (14 if case["grad"] else 4) * d * pairs * h}
    if case["kind"] == "rope":
        x = case["batch"] * case["tokens"] * (case["heads"] + case["kv"]) * case["d"]
        return {"bytes": (4 if case["grad"] else 2) * x * e + case["batch"] * case["tokens"] * 8, "flops": (30 if case["grad"] else 10) * x}
    n = sum(math.prod(s) for s in _shapes(case))
    return {"bytes": n * (3 * e + (16 if case["bits"] == 32 else 4)), "flops": (18 if case["bits"] == 32 else 60) * n}


# ---------------------------------------------------------------------------------------------------------------------
# float64
# ---------------------------------------------------------------------------------------------------------------------


def _exact_attn(case, st):
    n, m, group = case["queries"], case["keys"], case["heads"] // case["kv"]
    t = {k: st[k].detach().double() for k in ("q", "k", "v", "do")}
    o, dq = torch.zeros_like(t["q"]), torch.zeros_like(t["q"])
    dk, dv = torch.zeros_like(t["k"]), torch.zeros_like(t["k"])
    scale = case["d"] ** -0.5
    for b in range(case["batch"]):
        length = m if st["lengths"] is None else int(st["lengths"][b])
        first = m - n if st["starts"] is None else int(st["starts"][b])
        pos = torch.arange(first, first + n, device=DEV)
        live = torch.nonzero((pos >= 0) & (pos < length)).flatten()
        if not live.numel():
            continue
        keys = torch.arange(length, device=DEV)
        behind = pos[live, None] - keys
        hide = behind < 0
        if case["window"]:
            hide |= (behind >= case["window"]) & (keys >= case["sinks"])
        for h in range(case["heads"]):
            k, v, q = t["k"][b, :length, h // group], t["v"][b, :length, h // group], t["q"][b, live, h]
            s = (q @ k.t() * scale).masked_fill_(hide, -math.inf)
            p = torch.exp(s - torch.logsumexp(s, 1, keepdim=True))
            o[b, live, h] = p @ v
            if case["grad"]:
                g = t["do"][b, live, h]
                dp = g @ v.t()
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
                dq[b, live, h] = ds @ k
                dk[b, :length, h // group] += ds.t() @ q
                dv[b, :length, h // group] += p.t() @ g
    return (o, dq, dk, dv) if case["grad"] else o


def _exact_rope(case, st):
    rot, d, pos = case["rot"], case["d"], st["pos"].double()
    low = torch.arange(0, rot, 2, device=DEV) if case["interleaved"] else torch.arange(rot // 2, device=DEV)
    high = low + 1 if case["interleaved"] else low + rot // 2
    rate = torch.exp(torch.arange(rot // 2, device=DEV).double() * (-2 * math.log(10000.0) / rot))
    unit = torch.polar(torch.ones((), device=DEV, dtype=torch.float64), pos[:, :, None, None] * rate)

    def turned(u, by):
        z = torch.complex(u[..., low], u[..., high]) * by
        out = u.clone()
        out[..., low], out[..., high] = z.real, z.imag
        return out

    def one(x, w, g):
        x, w, g = x.detach().double(), w.detach().double(), g.double()
        c = x - x.mean(-1, keepdim=True) if case["norm"] == "layer" else x
        rstd = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS)
        hat = c * rstd
        y = turned(hat * w, unit)
        if not case["grad"]:
            return y, None, None
        du = turned(g, unit.conj())
        cw = du * w
        dx = cw - hat * (cw * hat).mean(-1, keepdim=True)
        if case["norm"] == "layer":
            dx = dx - cw.mean(-1, keepdim=True)
        return y, dx * rstd, (du * hat).reshape(-1, d).sum(0)

    q, dq, dqw = one(st["q"], st["qw"], st["dq"])
    k, dk, dkw = one(st["k"], st["kw"], st["dk"])
    return (q, k, dq, dk, dqw, dkw) if case["grad"] else (q, k)


def _exact_adamw(case, st):
    g = st["g"].double()
    norm = torch.linalg.vector_norm(g)
    if case["clip"] and float(norm) > 1.0:
        g = g / norm
    if case["bits"] == 32:
        m, v = st["m"].double(), st["v"].double()
    else:
        m, v = (torch.cat([c.double() * s.double().repeat_interleave(BLOCK)[:c.numel()] for c, s in st[k]]) for k in ("ms", "vs"))
        v = v ** 2
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g ** 2
    del g
    p = (1 - LR * DECAY) * st["p"].double()
    p -= LR / (1 - BETA1 ** STEP) * m / (torch.sqrt(v / (1 - BETA2 ** STEP)) + ADAM_EPS)
    if case["bits"] == 8:  # (the states that are kept are a choice among codes)
        return p, None, None, None, None
    return (p, m, v) + ((norm,) if case["clip"] else ())


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"attn": _exact_attn, "rope": _exact_rope, "adamw": _exact_adamw}[case["kind"]](case, st)
