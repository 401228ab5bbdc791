"""adamw_step and AdamW on the GPU: states in 32 bits against float64 within rounding bounds, states in 8 bits bit by bit against
the format's definition in numpy."""
import math

import numpy as np
import pytest
import torch

import psgd_pro_amd as P
from philox_ref import philox4x32_10

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.bfloat16]
SHAPES = [(1,), (7,), (3, 5), (), (256,), (257,), (64, 65), (4096,), (4097,), (130, 77), (0,), (1, 9000)]


@pytest.fixture(autouse=True)
def _lib(hip):
    return hip


def rnd(shape, seed, dtype=torch.float32, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def within(out, ref, bound, what=""):
    err = (out.double() - ref).abs()
    bad = ~(err <= bound + 1e-300)
    assert not bool(bad.any()), (what, int(bad.sum()), float((err / (bound + 1e-300)).nan_to_num(nan=9e9).max()))


def formula(p, g, m, v, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, coef=1.0):
    """((p, m, v), their bounds) in float64 from the values before."""
    store = U[p.dtype]
    p, g, m, v = (t.double() for t in (p, g, m, v))
    g = g * coef
    b1, b2 = betas
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    m_err = 5 * E * ((b1 * m).abs() + ((1 - b1) * g).abs())  # the constants, the gradient's factor, products and the sum
    v_err = 7 * E * v1 + 2.0 ** -148
    root, c = torch.sqrt(v1 / (1 - b2 ** step)), lr / (1 - b1 ** step)
    change = c * m1 / (root + eps)
    p1 = (1 - lr * weight_decay) * p - change
    # a root's relative error is half the square's, or its absolute error near zero
    root_err = torch.minimum(v_err / v1.clamp(min=1e-300), torch.ones_like(v1)) * root + 4 * E * root
    p_err = (c * m_err / (root + eps) + change.abs() * (root_err / (root + eps) + 8 * E) + 4 * E * (p.abs() + change.abs()) + store * p1.abs())
    return (p1, m1, v1), (p_err, m_err, v_err)


def tensors(dtype, seed=0, shapes=SHAPES):
    ps = [rnd(s, seed + 10 * i + 1, dtype) for i, s in enumerate(shapes)]
    gs = [rnd(s, seed + 10 * i + 2, dtype, std=0.1 * 10 ** -(i % 4)) for i, s in enumerate(shapes)]
    ms = [rnd(s, seed + 10 * i + 3, std=0.01) for i, s in enumerate(shapes)]
    vs = [rnd(s, seed + 10 * i + 4, std=0.1).square() for i, s in enumerate(shapes)]
    return ps, gs, ms, vs


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", [dict(step=1), dict(step=1000, lr=0.1, betas=(0.0, 0.5), eps=1e-3, weight_decay=0.5),
                                dict(step=3, lr=0.0), dict(step=2 ** 32, betas=(0.95, 0.0), weight_decay=-0.1)])
def test_32_bits_match_float64(dtype, kw):
    ps, gs, ms, vs = tensors(dtype)
    gs[4].zero_()
    vs[4][:100] = 0.0
    before = [[t.clone() for t in ts] for ts in (ps, ms, vs)]
    assert P.adamw_step(ps, gs, ms, vs, **kw) is None
    for i, (p, m, v) in enumerate(zip(*before)):
        refs, bounds = formula(p, gs[i], m, v, **kw)
        for name, t, r, e in zip("pmv", (ps[i], ms[i], vs[i]), refs, bounds):
            within(t, r, e, (name, i))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("max_norm", [1e-3, 1e6])
def test_clipping_by_the_norm_of_all(dtype, max_norm):
    ps, gs, ms, vs = tensors(dtype)
    before = [[t.clone() for t in ts] for ts in (ps, ms, vs)]
    norm = P.adamw_step(ps, gs, ms, vs, step=5, max_norm=max_norm)
    want = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    assert abs(float(norm) - want) <= 2 * E * want
    for i, (p, m, v) in enumerate(zip(*before)):
        refs, bounds = formula(p, gs[i], m, v, step=5, coef=min(1.0, max_norm / want))
        for t, r, e in zip((ps[i], ms[i], vs[i]), refs, bounds):
            within(t, r, e, i)


def test_norms_without_overflow_and_of_nothing():
    p, g, m, v = ([torch.full((5,), x, device=DEV)] for x in (1.0, 3e30, 0.0, 0.0))
    norm = P.adamw_step(p, g, m, v, step=1, max_norm=1.0)
    assert abs(float(norm) / (3e30 * math.sqrt(5)) - 1) < 4 * E
    assert torch.allclose(m[0], torch.full_like(m[0], 0.1 / math.sqrt(5)), rtol=1e-6)
    g[0].zero_()
    assert float(P.adamw_step(p, g, m, v, step=2, max_norm=1.0)) == 0.0 and p[0].isfinite().all()
    g[0][2] = math.nan
    assert math.isnan(float(P.adamw_step(p, g, m, v, step=3, max_norm=1.0))) and p[0].isnan().all()


# -- 8 bits -------------------------------------------------------------------------------------------------------------


def e4m3(codes):
    c = codes.astype(np.int64)
    ex, man = c >> 3 & 15, c & 7
    mag = np.where(ex > 0, 2.0 ** (ex - 7.0) * (1 + man / 8), 2.0 ** -6 * man / 8)
    return np.where(c >> 7, -mag, mag)


def unpack(codes, scales):
    s = np.where(scales == 0, 0.0, 2.0 ** (scales.astype(np.float64) - 127))
    return e4m3(codes) * np.repeat(s, 256)[:codes.size]


def pack(x, numbers, root):
    """The format from its definition: a block's scale, and of the codes around a magnitude the upper one where the share of the
    way to it plus the number's 65536th reaches one."""
    n, blocks = x.size, -(-x.size // 256)
    top = np.zeros(blocks * 256)
    top[:n] = np.abs(x)
    top = top.reshape(blocks, 256).max(1)
    mant, ex = np.frexp(top)  # top = mant 2^ex, mant in [.5, 1): the exponent field is ex - 1 + 127
    field = np.where(top > 0, np.maximum(ex - 1 + 127 + (mant > 0.875) - 8, 1), 0)
    mag = np.abs(x) / np.repeat(2.0 ** (field - 127.0), 256)[:n]
    grid = e4m3(np.arange(127))
    low = np.clip(np.searchsorted(grid, mag, side="right") - 1, 0, 126)
    step = np.where(low >= 8, 2.0 ** ((low >> 3) - 7.0) / 8, 2.0 ** -9)
    # bits below the code's lowest: 20 of them, those behind are rounded away only where a magnitude is subnormal in e4m3
    share = np.rint((mag - grid[low]) / step * 2 ** 20)
    code = low + (share + numbers * 16 >= 2 ** 20)
    if root:
        code = np.maximum(code, x > 0)
    return np.where(x < 0, code + 128, code).astype(np.uint8), field.astype(np.uint8)


def numbers(n, seed, step, tensor):
    out = np.empty((-(-n // 8), 8), dtype=np.int64)
    for b in range(out.shape[0]):
        w = philox4x32_10((b & 0xFFFFFFFF, b >> 32, step, tensor), (seed & 0xFFFFFFFF, seed >> 32))
        for c in range(8):
            out[b, c] = (w[c // 2] >> (16 * (c % 2))) & 0xFFFF
    return out.reshape(-1)[:n]


def step32(g, m, v, b1=0.9, b2=0.999):
    """m, v and its root in float32 arithmetic, each operation rounded."""
    f = np.float32
    g = g.astype(f)
    m = m.astype(f) * f(b1) + g * f(1 - b1)
    v = v.astype(f) * f(b2) + (g * g) * f(1 - b2)
    return m, v, np.sqrt(v)


def host(t):
    return t.view(torch.uint8).cpu().numpy()


@pytest.mark.parametrize("dtype", DTYPES)
def test_8_bits_match_their_definition(dtype):
    """Five steps over tensors of all sizes: codes and scales equal to those of the definition, parameters within rounding."""
    seed = 0x123456789ABCDEF
    ps, gs, _, _ = tensors(dtype, seed=5)
    gs[7][:300] *= 1e-12  # a block far below the others
    gs[8].zero_()
    ms, vs = ([P.adamw_state(p, 8) for p in ps] for _ in range(2))
    for step in range(1, 6):
        old = [(p.clone(), unpack(host(m[0]), host(m[1])), unpack(host(v[0]), host(v[1])) ** 2) for p, m, v in zip(ps, ms, vs)]
        P.adamw_step(ps, gs, ms, vs, step=step, seed=seed)
        for i, (p, m, v) in enumerate(old):
            g = gs[i].float().cpu().numpy().reshape(-1)
            m1, v1, root = step32(g, m, v)
            num = numbers(g.size, seed, step, i)
            for what, state, x, is_root in (("m", ms[i], m1, False), ("v", vs[i], root, True)):
                codes, scales = pack(x.astype(np.float64), num, is_root)
                assert np.array_equal(host(state[1]), scales), (what, i, step)
                assert np.array_equal(host(state[0]), codes), (what, i, step, int((host(state[0]) != codes).sum()))
            mt, vt = (torch.from_numpy(a.astype(np.float64)).to(DEV).view(p.shape) for a in (m, v))
            refs, bounds = formula(p, gs[i], mt, vt, step)
            within(ps[i], refs[0], bounds[0], (i, step))
        gs = [rnd(g.shape, 1000 + 17 * step + j, dtype, std=0.1 * 10 ** -(j % 5)) for j, g in enumerate(gs)]


def test_8_bits_lose_no_average():
    """A value between two codes has its own mean: 2^18 elements of one magnitude, a third of the way. The mean's deviation is
    the step's times sqrt(2/9) / 2^9; six of them."""
    n = 1 << 18
    p, g = [torch.zeros(n, device=DEV)], [torch.full((n,), 1.0 + 1 / 24, device=DEV)]
    g[0][::256] = 1.75  # the blocks' largest
    ms, vs = [P.adamw_state(p[0], 8)], [P.adamw_state(p[0], 8)]
    P.adamw_step(p, g, ms, vs, step=1, betas=(0.0, 0.0), seed=3)
    m = (ms[0][0].float() * ms[0][1].float().repeat_interleave(256))
    rest = torch.ones(n, dtype=torch.bool, device=DEV)
    rest[::256] = False
    assert set(m[rest].unique().tolist()) == {1.0, 1.125} and set(m[~rest].unique().tolist()) == {1.75}
    assert abs(float(m[rest].double().mean()) - (1 + 1 / 24)) < 6 * 0.125 * math.sqrt(2 / 9) / math.sqrt(n * 255 / 256)


def test_8_bits_forget():
    """Second moments decay though a step's change, a thousandth, is far below half a code: after 1000 steps without gradient
    e^-1 of them is left (their root's, on average over 2^16 elements; the rounding's variance adds a few hundredths)."""
    n = 1 << 16
    p, g = [torch.zeros(n, device=DEV)], [rnd((n,), 1)]
    ms, vs = [P.adamw_state(p[0], 8)], [P.adamw_state(p[0], 8)]
    P.adamw_step(p, g, ms, vs, step=1, betas=(0.9, 0.0), seed=1)
    value = lambda: (vs[0][0].float() * vs[0][1].float().repeat_interleave(256)).square().double().mean()  # noqa: E731
    start = float(value())
    g[0].zero_()
    for i in range(1000):
        P.adamw_step(p, g, ms, vs, step=2 + i, betas=(0.9, 0.999), seed=1)
    assert abs(float(value()) / start / math.exp(-1) - 1) < 0.1


@pytest.mark.parametrize("dtype", DTYPES)
def test_8_bits_at_the_ends_of_the_range(dtype):
    """Blocks of denormal, tiny and huge gradients; infinities and NaN make the block's states NaN and its parameters too."""
    shapes = [(256,)] * 6
    ps = [torch.ones(s, device=DEV, dtype=dtype) for s in shapes]
    gs = [torch.full(s, x, device=DEV, dtype=dtype) for s, x in zip(shapes, (1e-41, 1e-38, 1e-20, 1e18, 1.0, 1.0))]
    gs[4][5], gs[5][6] = math.inf, math.nan
    ms, vs = ([P.adamw_state(p, 8) for p in ps] for _ in range(2))
    for step in (1, 2):
        P.adamw_step(ps, gs, ms, vs, step=step, lr=1e-2, weight_decay=0.0)
        for i in range(4):
            assert ps[i].isfinite().all() and (ps[i] <= 1).all() and not ms[i][0].float().isnan().any()
    for i, hit in ((4, 5), (5, 6)):
        assert ms[i][1].float().isnan().all() and vs[i][1].float().isnan().all() and ps[i][hit].isnan()
    # A gradient of 1e-20 is nothing beside eps: m / (sqrt(v) + eps) is 1e-12. A steady one that is more than eps makes steps of lr,
    # the second within 14%: codes of both moments are up to an eighth off, which leaves m = .9 (.1 g) + .1 g within .059 of its
    # size and v = .999 (.001 g^2) + .001 g^2 within .135 (its root within .068); two roundings of a bfloat16 below 1 are 2^-9 each.
    assert bool((ps[2] == 1).all())
    assert bool(((ps[3].double() - 0.98).abs() <= 0.14 * 0.01 + (2 * 2.0 ** -9 if dtype == torch.bfloat16 else 1e-6)).all())


# -- layouts --------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", DTYPES)
def test_views_on_odd_boundaries_leave_their_neighbours(bits, dtype):
    """Tensors, gradients and states one after the other on no boundary, with guards between: the same bits as tensors of their
    own, and the guards stay."""
    sizes = [1, 3, 255, 256, 257, 4099, 777]
    flat = rnd((sum(sizes) + 5 * len(sizes),), 1, dtype)
    fg = rnd(flat.shape, 2, dtype)
    fm, fv = ([P.adamw_state(flat, 32) for _ in range(2)] if bits == 32 else
              [torch.zeros(flat.numel(), device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)])
    fs = [torch.zeros(200, device=DEV, dtype=torch.uint8).view(torch.float8_e8m0fnu) for _ in range(2)]
    keep = flat.clone()
    ps, gs, ms, vs, at, sc, mask = [], [], [], [], 3, 1, torch.ones(flat.numel(), dtype=torch.bool, device=DEV)
    for n in sizes:
        k = -(-n // 256)
        ps.append(flat[at:at + n])
        gs.append(fg[at:at + n])
        for out, f, s in ((ms, fm, fs[0]), (vs, fv, fs[1])):
            out.append(f[at:at + n] if bits == 32 else (f[at:at + n], s[sc:sc + k]))
        mask[at:at + n] = False
        at, sc = at + n + 5, sc + k + 1
    own = [p.clone() for p in ps], [g.clone() for g in gs], [P.adamw_state(p, bits) for p in ps], [P.adamw_state(p, bits) for p in ps]
    for step in (1, 2):
        P.adamw_step(ps, gs, ms, vs, step=step, seed=9)
        P.adamw_step(*own, step=step, seed=9)
    assert all(torch.equal(a, b) for a, b in zip(ps, own[0])) and torch.equal(flat[mask], keep[mask])
    for views, mine, f in ((ms, own[2], fm), (vs, own[3], fv)):
        for a, b in zip(views, mine):
            assert torch.equal(a, b) if bits == 32 else all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))
        assert not (f if bits == 32 else f.view(torch.uint8))[mask].any()


def test_hundreds_of_tensors_of_both_dtypes():
    """More tensors than a launch takes, dtypes in turn, gradients that are not contiguous: each as by itself."""
    n = 300
    ps = [rnd((5 + i % 7, 11 + i % 3), i, DTYPES[i % 2]) for i in range(n)]
    gs = [rnd((p.shape[1], p.shape[0]), 1000 + i, p.dtype).t() if i % 3 else rnd((1, 1), i, p.dtype).expand(p.shape) for i, p in enumerate(ps)]
    ms, vs = ([P.adamw_state(p) for p in ps] for _ in range(2))
    alone = [(p.clone(), P.adamw_state(p), P.adamw_state(p)) for p in ps]
    P.adamw_step(ps, gs, ms, vs, step=4, lr=0.01)
    for i, (p, m, v) in enumerate(alone):
        P.adamw_step([p], [gs[i]], [m], [v], step=4, lr=0.01)
        assert torch.equal(p, ps[i]) and torch.equal(m, ms[i]) and torch.equal(v, vs[i])


def test_a_tensor_beyond_32_bits():
    """2^32 + 5 elements of bfloat16 with 8-bit states: the last ones as those of a short tensor at the same place of a block."""
    n = (1 << 32) + 5
    p = torch.ones(n, device=DEV, dtype=torch.bfloat16)
    g = torch.zeros(n, device=DEV, dtype=torch.bfloat16)
    g[-5:] = torch.tensor([1, -2, 3, -4, 5.0], device=DEV)
    m, v = P.adamw_state(p, 8), P.adamw_state(p, 8)
    norm = P.adamw_step([p], [g], [m], [v], step=1, lr=0.5, weight_decay=0.0, max_norm=1e9)
    assert abs(float(norm) - math.sqrt(55)) < 1e-5
    assert p[-6:].tolist() == [1.0, 0.5, 1.5, 0.5, 1.5, 0.5] and bool((p[:-5] == 1).all())
    assert not bool(m[0].view(torch.uint8)[:-5].any()) and m[1].view(torch.uint8)[-1] != 0 and not bool(m[1].view(torch.uint8)[:-1].any())


# -- the optimizer --------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_is_the_function(bits):
    shapes = [(33, 20), (20,), ()]
    ps = [rnd(s, i).requires_grad_() for i, s in enumerate(shapes)]
    copies = [p.detach().clone() for p in ps]
    opt = P.AdamW(ps, lr_params=0.01, betas=(0.8, 0.95), weight_decay=0.1, max_norm=0.5, state_bits=bits, seed=77)
    ms, vs = ([P.adamw_state(p, bits) for p in copies] for _ in range(2))
    for step in range(1, 4):
        gs = [rnd(s, 100 * step + i) for i, s in enumerate(shapes)]
        opt.step_math(gs)
        norm = P.adamw_step(copies, gs, ms, vs, step=step, lr=0.01, betas=(0.8, 0.95), weight_decay=0.1, max_norm=0.5, seed=77)
        assert float(opt.norm) == float(norm)
    assert all(torch.equal(a.detach(), b) for a, b in zip(ps, copies))
    for i in range(3):
        m, v = opt.moments(i)
        if bits == 32:
            assert torch.equal(m, ms[i]) and torch.equal(v, vs[i])
        else:
            want = unpack(host(vs[i][0]), host(vs[i][1])) ** 2
            assert m.shape == ps[i].shape and np.allclose(v.cpu().numpy().reshape(-1), want, rtol=1e-6)


@pytest.mark.parametrize("bits", [8, 32])
def test_closure_and_state_dict(bits):
    w = rnd((40, 30), 1).requires_grad_()
    opt = P.AdamW(w, state_bits=bits, seed=5)
    loss = lambda: ((w ** 2).sum(), "told")  # noqa: E731
    for _ in range(3):
        out = opt.step(loss)
    assert out[1] == "told"
    saved, at = opt.state_dict(), w.detach().clone()
    for _ in range(2):
        opt.step(loss)
    end = w.detach().clone()
    again = at.clone().requires_grad_()
    other = P.AdamW([again], lr_params=9.0, state_bits=bits)
    other.load_state_dict(saved)
    for _ in range(2):
        other.step_math([2 * again.detach()])
    assert torch.equal(again.detach(), end)
    with pytest.raises(ValueError, match="bits"):
        P.AdamW([again], state_bits=40 - bits).load_state_dict(saved)
    with pytest.raises(ValueError, match="shape"):
        P.AdamW([rnd((41, 30), 1).requires_grad_()], state_bits=bits).load_state_dict(saved)


def test_a_step_between_forward_and_backward_is_noticed():
    w = rnd((4, 4), 1).requires_grad_()
    opt = P.AdamW(w)
    loss = (w ** 2).sum()
    P.AdamW(w)  # (making one changes nothing)
    torch.autograd.grad(loss, w, retain_graph=True)
    opt.step_math([rnd((4, 4), 2)])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, w)


def test_captures_are_refused():
    ps, gs, ms, vs = tensors(torch.float32, shapes=[(5,)])
    P.adamw_step(ps, gs, ms, vs, step=1)
    torch.cuda.synchronize()
    x = torch.zeros(4, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="captured"):
            P.adamw_step(ps, gs, ms, vs, step=2)
    graph.replay()
    torch.cuda.synchronize()
    assert float(x[0]) == 1.0


@pytest.mark.parametrize("kw", [dict(step=0), dict(step=1, lr=math.nan), dict(step=1, weight_decay=math.inf), dict(step=1, betas=(1.0, 0.9)),
                                dict(step=1, betas=(0.9, -0.1)), dict(step=1, eps=-1e-8), dict(step=1, max_norm=0.0), dict(step=1, max_norm=math.nan)])
def test_refusals_of_numbers(kw):
    with pytest.raises(ValueError):
        P.adamw_step(*tensors(torch.float32, shapes=[(5,)]), **kw)


def test_refusals_of_tensors():
    def call(**kw):
        ps, gs, ms, vs = tensors(torch.float32, shapes=[(6, 4), (5,)])
        a = dict(p=ps, g=gs, m=ms, v=vs)
        for k, f in kw.items():
            f(a[k])
        P.adamw_step(a["p"], a["g"], a["m"], a["v"], step=1)

    def put(i, t):
        return lambda ts: ts.__setitem__(i, t(ts[i]))

    call()
    for bad in (dict(p=put(0, lambda t: t.t())), dict(p=put(0, lambda t: t.cpu())), dict(p=put(1, lambda t: t.view(5, 1))), dict(g=put(0, lambda t: t.bfloat16())),
                dict(g=put(0, lambda t: t.t())), dict(g=lambda ts: ts.pop()), dict(m=put(0, lambda t: t.bfloat16())), dict(m=put(1, lambda t: t[:4])),
                dict(v=put(0, lambda t: t.t())), dict(v=put(0, lambda t: P.adamw_state(t, 8))), dict(m=lambda ts: ts.pop()), dict(g=put(1, lambda t: None)),
                dict(p=lambda ts: ts.__setitem__(1, ts[0].view(-1)[:5]))):
        with pytest.raises(RuntimeError):
            call(**bad)
    with pytest.raises(TypeError):
        call(p=put(0, lambda t: t.double()))
    with pytest.raises(RuntimeError, match="no parameters"):
        P.adamw_step([], [], [], [], step=1)
    with pytest.raises(ValueError):
        P.AdamW([torch.zeros(3, device=DEV)])
    with pytest.raises(ValueError):
        P.AdamW([torch.zeros(3, device=DEV, requires_grad=True)], state_bits=16)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_state_given_twice_is_refused(bits):
    ps, gs = [[torch.ones(300, device=DEV) for _ in range(2)] for _ in range(2)]
    ms, vs = [[P.adamw_state(p, bits) for p in ps] for _ in range(2)]
    for m, v in ((ms, ms), ([ms[0], ms[0]], vs), (ms, [vs[0], vs[0]])):
        with pytest.raises(RuntimeError, match="twice"):
            P.adamw_step(ps, gs, m, v, step=1)
    assert all(bool((p == 1).all()) for p in ps)
    if bits == 8:
        with pytest.raises(RuntimeError, match="twice"):
            P.adamw_step(ps, gs, [ms[0], (ms[1][0], ms[0][1])], vs, step=1)
    P.adamw_step(ps, gs, ms, vs, step=1)
