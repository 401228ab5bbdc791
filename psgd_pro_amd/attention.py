"""Attention of a transformer's block on the HIP kernels (include/psgdk.h, level 3).

    qk_norm_rope       norms of queries and keys for each head and their rotation by position, one pass
    window_attention   softmax attention with grouped heads, a sliding window and first tokens that stay visible

CUDA (HIP) tensors in float32 or bfloat16, on torch's current stream, differentiable once through autograd. No counterparts in
the reference, which leaves the model to torch.
"""
import ctypes as C
import math

import torch

from . import _lib as L
from .train import _NORMS, _check, _once, _ptr, _run, _run_ws, _wants_grad

__all__ = ["qk_norm_rope", "window_attention"]

_MAX_STRIDE = 1 << 21  # of tokens, and of queries' heads, in elements


def _heads(t, keys=False):
    """(psgdk_heads_t of t, the tensor it points to): t itself where its rows are aligned, else a copy. Heads of keys may lie any
    distance apart (a cache of each head's tokens), those of queries are rows of one tile."""
    unit = 16 // t.element_size()
    sb, sn, sh, sd = t.stride()
    if (sd != 1 or t.data_ptr() % 16 or sb % unit or sn % unit or sh % unit or sn > _MAX_STRIDE
            or (not keys and sh * max(t.shape[2], 128) > _MAX_STRIDE * 128)):
        t = t.clone(memory_format=torch.contiguous_format)
        sb, sn, sh, _ = t.stride()
    return L.Heads(t.data_ptr(), sb, sn, sh), t


def _attn_block(q, k, v, lengths, starts, o, lse, rest, opt):
    """psgdk_window_attention_t of the inputs, and the (possibly copied) tensors it points to."""
    window, sinks, scale = opt
    a = L.WindowAttention(q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3], L.dtype_code(q.dtype), window,
                          sinks, scale)
    (a.q, q), (a.k, k), (a.v, v) = _heads(q), _heads(k, True), _heads(v, True)
    a.lengths, a.starts, a.o, a.lse, a.o_rest = _ptr(lengths), _ptr(starts), o.data_ptr(), _ptr(lse), _ptr(rest)
    return a, (q, k, v)


def _attn_forward(q, k, v, lengths, starts, opt, stats):
    o = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    lse = torch.empty(q.shape[:3], device=q.device, dtype=torch.float32) if stats else None
    rest = torch.empty_like(o) if stats and q.dtype == torch.bfloat16 else None
    if not q.numel():
        return o, lse, rest
    if not k.numel():  # no key to see
        return o.zero_(), lse, rest
    a, keep = _attn_block(q, k, v, lengths, starts, o, lse, rest, opt)
    _run_ws(q, L.lib().psgdk_window_attention, C.byref(a))
    return o, lse, rest


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, starts, opt):
        o, lse, rest = _attn_forward(q, k, v, lengths, starts, opt, True)
        ctx.opt = opt
        ctx.save_for_backward(q, k, v, lengths, starts, o, lse, rest)
        return o

    @staticmethod
    def backward(ctx, do):
        _once()
        q, k, v, lengths, starts, o, lse, rest = ctx.saved_tensors
        outs = [torch.empty(t.shape, device=t.device, dtype=t.dtype) if need else None
                for t, need in zip((q, k, v), ctx.needs_input_grad)]
        if not q.numel() or not k.numel():
            for t in outs:
                if t is not None:
                    t.zero_()
            return (*outs, None, None, None)
        a, keep = _attn_block(q, k, v, lengths, starts, o, lse, rest, ctx.opt)
        g = L.WindowAttentionGrads()
        g.dout, do = _heads(do)
        g.dq, g.dk, g.dv = (_ptr(t) for t in outs)
        _run_ws(q, L.lib().psgdk_window_attention_backward, C.byref(a), C.byref(g))
        return (*outs, None, None, None)


def window_attention(q, k, v, *, window=None, sinks=0, scale=None, lengths=None, starts=None):
    """Causal attention: q (batch, n, heads, d), k and v (batch, m, kv_heads, d), heads a multiple of kv_heads (query head h takes
    the keys of head h // (heads // kv_heads)), d a multiple of 8 up to 128; any strides (rows that are not 16-byte aligned are
    copied). Returns (batch, n, heads, d).

    Query i of sequence b is at position p = starts[b] + i, and sees key j where 0 <= p < lengths[b], j <= p, and (with a window)
    p - j < window or j < sinks. lengths and starts are int64 tensors (batch,); absent, every sequence has m tokens and its
    queries are the last n of them, so that

        window_attention(q, k, v)                                    trains on whole sequences,
        window_attention(q, k, v, lengths=n_tokens)                  on a batch padded on the right,
        window_attention(q, kc, vc, lengths=n_tokens, starts=n_tokens - n)    reads the caches kc, vc of m places for the
                                                                     last n tokens of each sequence.

    A query that sees nothing has output 0 and no gradient; keys and values from lengths[b] on, and queries and gradients of
    positions outside the sequence, may hold anything. Within a sequence values are taken to be finite: an infinity or NaN may
    reach queries that do not see it. bfloat16 probabilities (where a key head has more than 64 queries), and backward the
    scores' gradients, are rounded before the second products. Two runs give the same bits. scale: 1 / sqrt(d) if not given. Differentiable in q, k and v."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check(t, name, None if t is q else q)
        if t.dim() != 4 or t.dtype != q.dtype:
            raise RuntimeError(f"{name}: (batch, tokens, heads, d) in {q.dtype} expected, got {tuple(t.shape)} in {t.dtype}")
    b, n, h, d = q.shape
    if k.shape != v.shape or k.shape[0] != b or k.shape[3] != d:
        raise RuntimeError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: batch and d of q, k and v alike expected")
    if not h or not k.shape[2] or h % k.shape[2]:
        raise RuntimeError(f"{h} query heads: a multiple of the {k.shape[2]} key heads expected")
    if not 8 <= d <= 128 or d % 8:
        raise RuntimeError(f"d = {d}: a multiple of 8 up to 128 expected")
    if window is not None and not window >= 1:
        raise ValueError(f"window = {window}: at least 1, or None")
    if not sinks >= 0:
        raise ValueError(f"sinks = {sinks}: must be >= 0")
    scale = 1 / math.sqrt(d) if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale = {scale}: must be positive")
    tell = []
    for name, t in (("lengths", lengths), ("starts", starts)):
        if t is not None and (not isinstance(t, torch.Tensor) or t.dtype != torch.int64 or t.device != q.device or t.shape != (b,)):
            raise RuntimeError(f"{name}: an int64 tensor ({b},) on {q.device} expected")
        tell.append(t if t is None else t.contiguous())
    opt = (min(int(window), 1 << 40) if window is not None else 0, min(int(sinks), 1 << 40), scale)
    if _wants_grad(q, k, v):
        return _WindowAttention.apply(q, k, v, *tell, opt)
    return _attn_forward(q, k, v, *tell, opt, False)[0]


# -- qk_norm_rope -----------------------------------------------------------------------------------------------------------


def _dense(t):
    """(psgdk_heads_t of t, the tensor it points to): any strides, a head's elements one after the other."""
    if t.stride(3) != 1 and t.shape[3] > 1:
        t = t.contiguous()
    return L.Heads(t.data_ptr(), *t.stride()[:3]), t


def _rope_block(q, k, qw, kw, pos, opt):
    """psgdk_qk_norm_rope_t of the inputs, and the (possibly copied) tensors it points to."""
    norm, eps, theta, rot, interleaved = opt
    w = [t if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0) else t.clone(memory_format=torch.contiguous_format)
         for t in (qw, kw)]
    some = qw if qw is not None else kw
    a = L.QkNormRope(q.shape[0], q.shape[1], q.shape[2], 0 if k is None else k.shape[2], q.shape[3], rot, L.dtype_code(q.dtype),
                     L.F32 if some is None else L.dtype_code(some.dtype), norm, interleaved, eps, theta, _ptr(pos),
                     0 if pos is None or pos.dim() == 1 else pos.shape[1])
    a.q, q = _dense(q)
    if k is not None:
        a.k, k = _dense(k)
    a.q_w, a.k_w = (_ptr(t) for t in w)
    return a, (q, k, w)


def _rope_forward(q, k, qw, kw, pos, opt):
    a, keep = _rope_block(q, k, qw, kw, pos, opt)
    qo = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    ko = None if k is None else torch.empty(k.shape, device=q.device, dtype=q.dtype)
    if qo.numel():
        _run(q, L.lib().psgdk_qk_norm_rope, C.byref(a), qo.data_ptr(), _ptr(ko))
    return qo, ko


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, qw, kw, pos, opt):
        ctx.set_materialize_grads(False)
        ctx.opt = opt
        ctx.save_for_backward(q, k, qw, kw, pos)
        return _rope_forward(q, k, qw, kw, pos, opt)

    @staticmethod
    def backward(ctx, dqo, dko):
        _once()
        q, k, qw, kw, pos = ctx.saved_tensors
        outs = [torch.empty(t.shape, device=t.device, dtype=t.dtype) if t is not None and need else None
                for t, need in zip((q, k, qw, kw), ctx.needs_input_grad)]
        if not q.numel():
            for t in outs:
                if t is not None:
                    t.zero_()
            return (*outs, None, None)
        a, keep = _rope_block(q, k, qw, kw, pos, ctx.opt)
        g = L.QkNormRopeGrads()
        if dqo is not None:
            g.dqo, dqo = _dense(dqo)
        if dko is not None:
            g.dko, dko = _dense(dko)
        g.dq, g.dk, g.dqw, g.dkw = (_ptr(t) for t in outs)
        _run_ws(q, L.lib().psgdk_qk_norm_rope_backward, C.byref(a), C.byref(g))
        return (*outs, None, None)


def qk_norm_rope(q, k=None, *, norm="rms", q_weight=None, k_weight=None, eps=1e-6, positions=None, theta=10000.0,
                 rotary_dim=None, interleaved=False):
    """(q', k'): queries q (batch, n, heads, d) and keys k (batch, n, kv_heads, d; None: k' is None) normalised over each head's
    d, times their weights (d,), and rotated by their tokens' positions, in one pass.

        u = N(x) * w;  pair (a, b) of u becomes (a cos t - b sin t, b cos t + a sin t),  t = p theta^(-2 i / rotary_dim)

    norm: "rms" (v / sqrt(mean v^2 + eps)), "layer" ((v - mean) / sqrt(var + eps)) or None (no weights then); weights may be
    absent and may be float32 beside bfloat16 inputs. Pair i of the first rotary_dim elements (d if not given; even) is
    (i, i + rotary_dim / 2), or (2 i, 2 i + 1) where interleaved; the elements behind are not rotated. positions: int64 (n,) or
    (batch, n); a token's index in its sequence if not given. Angles are right to float32's rounding up to position 2^24 and to
    |p| 2^-48 beyond, and add up as positions do. d is even and up to 512, q and k may have any strides; q' and k' are
    contiguous. Differentiable in q, k and the weights."""
    if norm not in _NORMS:
        raise ValueError(f"norm = {norm!r}: 'rms', 'layer' or None")
    _check(q, "q")
    for name, t in (("q", q), ("k", k)):
        if t is None:
            continue
        _check(t, name, q)
        if t.dim() != 4 or t.dtype != q.dtype or t.shape[:2] != q.shape[:2] or t.shape[3] != q.shape[3]:
            raise RuntimeError(f"{name}: (batch, n, heads, d) in {q.dtype} expected, batch, n and d as q's, got {tuple(t.shape)} in "
                               f"{t.dtype}")
        if not t.shape[2]:
            raise RuntimeError(f"{name}: at least one head expected")
    d = q.shape[3]
    if not 2 <= d <= 512 or d % 2:
        raise RuntimeError(f"d = {d}: even and up to 512 expected")
    for name, t, of in (("q_weight", q_weight, q), ("k_weight", k_weight, k)):
        if t is None:
            continue
        _check(t, name, q)
        if norm is None or of is None:
            raise ValueError(f"{name}: " + ("the norm None has none" if norm is None else "needs k"))
        if t.shape != (d,) or (q_weight is not None and t.dtype != q_weight.dtype):
            raise RuntimeError(f"{name}: shape ({d},) expected, and one dtype for both weights; got {tuple(t.shape)} in {t.dtype}")
    rot = d if rotary_dim is None else int(rotary_dim)
    if not 0 <= rot <= d or rot % 2:
        raise ValueError(f"rotary_dim = {rotary_dim}: even and in 0..{d}")
    if not (theta >= 1 and math.isfinite(theta)):
        raise ValueError(f"theta = {theta}: must be at least 1")
    if not eps >= 0:
        raise ValueError(f"eps = {eps}: must be >= 0")
    if positions is not None:
        if (not isinstance(positions, torch.Tensor) or positions.dtype != torch.int64 or positions.device != q.device
                or tuple(positions.shape) not in (tuple(q.shape[1:2]), tuple(q.shape[:2]))):
            raise RuntimeError(f"positions: an int64 tensor ({q.shape[1]},) or ({q.shape[0]}, {q.shape[1]}) on {q.device} expected")
        positions = positions.contiguous()
    opt = (_NORMS[norm], float(eps), float(theta), rot, int(bool(interleaved)))
    if _wants_grad(q, k, q_weight, k_weight):
        return _QkNormRope.apply(q, k, q_weight, k_weight, positions, opt)
    return _rope_forward(q, k, q_weight, k_weight, positions, opt)
