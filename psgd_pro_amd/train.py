"""Operators of the training step in front of the optimizer, on the HIP kernels (include/psgdk.h, level 3).

    linear_cross_entropy   the loss of a language model's head from its inputs and vocabulary matrix, logits never kept
    residual_norm          the residual sum between two blocks of a transformer with its norms, gate, scale and dropout
    dropout                dropout from the library's counter-based generator, mask never stored

All take CUDA (HIP) tensors in float32 or bfloat16, run on torch's current stream and differentiate once through
autograd (not in forward mode, which is refused). No counterparts in the reference, which leaves the model to torch.
"""
import ctypes as C

import torch
from torch.autograd import forward_ad
from . import _lib as L

__all__ = ["dropout", "linear_cross_entropy", "residual_norm"]

_NORMS = {None: L.NORM_NONE, "rms": L.NORM_RMS, "layer": L.NORM_LAYER}


_DTYPES = (torch.float32, torch.bfloat16)


def _check(t, name, like=None):
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in _DTYPES and (like is None or t.get_device() == like.get_device()):
        return
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"{name}: psgd_pro_amd ops take CUDA (HIP) tensors; got " +
                           (f"a tensor on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__))
    if t.dtype not in _DTYPES:
        raise RuntimeError(f"{name}: float32 or bfloat16 expected, got {t.dtype}")
    raise RuntimeError(f"{name}: on {t.device}, the input is on {like.device}")


def _rows(t):
    """(r, ld): t as rows of its last dimension, contiguous inside a row, ld elements from one to the next; r is t itself
    where its rows lie one after the other, a view where its strides allow, else a copy."""
    d = t.shape[-1]
    if t.is_contiguous():
        return t, d
    r = t.reshape(-1, d) if t.dim() != 2 else t
    if (d > 1 and r.stride(1) != 1) or (r.shape[0] > 1 and r.stride(0) < d):
        r = r.contiguous()
    return r, r.stride(0) if r.shape[0] > 1 else d


def _run(t, fn, *args):
    """fn(*args, stream) on t's device and its current stream."""
    i = t.get_device()
    if i == torch._C._cuda_getDevice():
        L.check(fn(*args, torch._C._cuda_getCurrentRawStream(i)))
    else:
        with torch.cuda.device(i):
            L.check(fn(*args, torch._C._cuda_getCurrentRawStream(i)))


def _run_ws(t, fn, *args):
    """fn(*args, workspace, its size, stream): the size asked for first, the workspace back with torch's allocator after."""
    size = C.c_size_t(0)
    L.check(fn(*args, None, C.byref(size), None))
    ws = torch.empty(max(size.value, 256), dtype=torch.uint8, device=t.device)
    _run(t, fn, *args, ws.data_ptr(), C.byref(size))


def _once():
    """The backward functions' outputs have no graph of their own."""
    if torch.is_grad_enabled():
        raise RuntimeError("psgd_pro_amd ops differentiate once: no create_graph through them")


def _wants_grad(*ts):
    # (the plain call would leave a tangent behind without a word, and grad mode says nothing about forward mode)
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled() and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise RuntimeError("psgd_pro_amd ops have no forward-mode derivatives")
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _seed(seed, p):
    """The generator's 64-bit key; with no seed given, one drawn from torch's CPU generator (as KronWhiten's)."""
    if seed is None:
        return int(torch.randint(2 ** 62, ())) if p else 0
    return int(seed) & (2 ** 64 - 1)


def _check_p(p):
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p = {p}: must be in 0..1")


# -- dropout ----------------------------------------------------------------------------------------------------------


def _dropout_call(x, p, seed, stream):
    y = x.new_empty(x.shape)
    n, d = x.numel(), x.shape[-1]
    if n:
        r, ld = _rows(x)
        _run(x, L.lib().psgdk_dropout, n // d, d, L.dtype_code(x.dtype), r.data_ptr(), ld, y.data_ptr(), d, p, seed, stream)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, stream):
        ctx.args = p, seed, stream
        return _dropout_call(x, p, seed, stream)

    @staticmethod
    def backward(ctx, g):
        _once()
        return _dropout_call(g, *ctx.args), None, None, None


def dropout(x, p, *, seed=None, stream=0):
    """x with each element set to 0 with probability p and the others scaled by 1 / (1 - p).

    p is taken in steps of 2^-16: with t = round(65536 p), element (i, c) of x seen as rows of its last dimension d is
    kept where the 16-bit number c % 8 of block i ceil(d / 8) + c / 8 of the Philox4x32-10 sequence of (seed, stream) is
    at least t, and scaled by 65536 / (65536 - t). The mask is made again in the backward pass. The same (seed, stream)
    and shape give the same mask; seed None draws one from torch's CPU generator. Give each call of a step its own
    stream (a layer's number, say) under one seed."""
    _check(x, "x")
    _check_p(p)
    if x.dim() == 0:
        raise RuntimeError("x: at least one dimension expected")
    seed, stream = _seed(seed, p), int(stream) & (2 ** 64 - 1)
    if _wants_grad(x):
        return _Dropout.apply(x, float(p), seed, stream)
    return _dropout_call(x, float(p), seed, stream)


# -- residual_norm ----------------------------------------------------------------------------------------------------


def _ptr(t):
    return None if t is None else t.data_ptr()


def _res_block(x, f, gate, pw, pb, qw, qb, opt):
    """psgdk_residual_norm_t of the inputs, and the (possibly copied) tensors it points to."""
    pre, post, scale, eps, p, seed, stream, gate_rows = opt
    d = x.shape[-1]
    w = [t if t is None or t.is_contiguous() else t.contiguous() for t in (pw, pb, qw, qb)]
    a = L.ResidualNorm()
    a.rows, a.d = x.numel() // max(d, 1), d
    a.dtype = L.dtype_code(x.dtype)
    a.pre, a.post, a.eps, a.scale, a.p, a.seed, a.stream_id, a.gate_rows = pre, post, eps, scale, p, seed, stream, gate_rows
    xr, a.ldx = _rows(x)
    a.x = xr.data_ptr()
    keep = [xr, w]
    if f is not None:
        fr, a.ldf = _rows(f)
        a.f = fr.data_ptr()
        keep.append(fr)
    if gate is not None:
        gr, a.ldgate = _rows(gate)
        a.gate, a.gate_dtype = gr.data_ptr(), L.dtype_code(gate.dtype)
        keep.append(gr)
    a.pre_w, a.pre_b, a.post_w, a.post_b = (_ptr(t) for t in w)
    some = next((t for t in w if t is not None), None)
    a.w_dtype = L.F32 if some is None else L.dtype_code(some.dtype)
    return a, keep


def _res_forward(x, f, gate, pw, pb, qw, qb, opt, stats):
    a, keep = _res_block(x, f, gate, pw, pb, qw, qb, opt)
    y = x.new_empty(x.shape) if f is not None else None
    h = x.new_empty(x.shape) if opt[0] else None
    st = torch.empty(a.rows, 4, device=x.device, dtype=torch.float32) if stats else None
    a.y, a.ldy, a.h, a.ldh, a.stats = _ptr(y), a.d, _ptr(h), a.d, _ptr(st)
    if x.numel() and (y is not None or h is not None):
        _run(x, L.lib().psgdk_residual_norm, C.byref(a))
    return y, h, st


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, gate, pw, pb, qw, qb, opt):
        ctx.set_materialize_grads(False)
        y, h, st = _res_forward(x, f, gate, pw, pb, qw, qb, opt, True)
        ctx.opt = opt
        ctx.save_for_backward(x, f, gate, pw, pb, qw, qb, st)
        if y is None:
            y = x.view_as(x)
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        _once()
        x, f, gate, pw, pb, qw, qb, st = ctx.saved_tensors
        need = ctx.needs_input_grad
        a, keep = _res_block(x, f, gate, pw, pb, qw, qb, ctx.opt)
        a.stats = _ptr(st)
        g = L.ResidualNormGrads()
        if dy is not None:
            dy, g.lddy = _rows(dy)
            g.dy = dy.data_ptr()
        if dh is not None:
            dh, g.lddh = _rows(dh)
            g.dh = dh.data_ptr()
        outs = [None] * 8
        for k, (name, like) in enumerate((("dx", x), ("df", f), ("dgate", gate), ("dpre_w", pw), ("dpre_b", pb),
                                          ("dpost_w", qw), ("dpost_b", qb))):
            if like is None or not need[k]:
                continue
            outs[k] = like.new_empty(like.shape)
            setattr(g, name, outs[k].data_ptr())
            if k < 3:
                setattr(g, "ld" + name, like.shape[-1])
        if not x.numel():
            for t in outs:
                if t is not None:
                    t.zero_()
        else:
            _run_ws(x, L.lib().psgdk_residual_norm_backward, C.byref(a), C.byref(g))
        return tuple(outs)


def _gate_rows(gate, x):
    """Rows of the gate: its leading dimensions are x's first ones, then ones (fewer dimensions: ones in front)."""
    lead, xs = tuple(gate.shape[:-1]), tuple(x.shape[:-1])
    bad = f"gate: shape {tuple(gate.shape)} does not go with {tuple(x.shape)} (its last dimension, and its first ones or ones)"
    if gate.dim() == 0 or gate.shape[-1] != x.shape[-1] or len(lead) > len(xs):
        raise RuntimeError(bad)
    lead = (1,) * (len(xs) - len(lead)) + lead
    n = 0
    while n < len(xs) and lead[n] == xs[n]:
        n += 1
    if any(v != 1 for v in lead[n:]):
        raise RuntimeError(bad)
    rows = 1
    for v in lead:
        rows *= v
    return rows


def residual_norm(x, f=None, *, pre="rms", post=None, pre_weight=None, pre_bias=None, post_weight=None, post_bias=None,
                  gate=None, scale=1.0, eps=1e-6, p=0.0, seed=None, stream=0):
    """(y, h): the residual sum after a block of a transformer and the next block's normalised input, in one pass.

        u = Npost(f);  b = dropout(u, p, seed, stream);  y = x + scale * gate * b;  h = Npre(y)

    x is the residual stream (any shape, norms over the last dimension), f the block's output (None: y is x, as in front
    of the first block). pre and post choose the norms: "rms" (v / sqrt(mean v^2 + eps) * weight), "layer"
    ((v - mean) / sqrt(var + eps) * weight + bias) or None (pre None: h is None); weights and biases may be absent and may
    be float32 beside bfloat16 activations. gate has x's last dimension, and in front of it x's first dimensions followed
    by ones: (d,) scales channels, (batch, 1, d) each sequence's, x's own shape every element. h is made from the sum
    before its rounding. Differentiable in x, f, gate and the norms' parameters."""
    _check(x, "x")
    _check_p(p)
    if x.dim() == 0:
        raise RuntimeError("x: at least one dimension expected")
    d = x.shape[-1]
    for name, kind in (("pre", pre), ("post", post)):
        if kind not in _NORMS:
            raise ValueError(f"{name} = {kind!r}: 'rms', 'layer' or None")
    if f is None and (post is not None or gate is not None or p):
        raise ValueError("post, gate and p need f")
    if pre is None and f is None:
        raise ValueError("nothing to compute: neither f nor a norm")
    if f is not None:
        _check(f, "f", x)
        if f.shape != x.shape or f.dtype != x.dtype:
            raise RuntimeError(f"f: {tuple(f.shape)} {f.dtype} expected as x, {tuple(x.shape)} {x.dtype}")
    par = (pre_weight, pre_bias, post_weight, post_bias)
    for name, t, kinds, kind in (("pre_weight", pre_weight, ("rms", "layer"), pre), ("pre_bias", pre_bias, ("layer",), pre),
                                 ("post_weight", post_weight, ("rms", "layer"), post),
                                 ("post_bias", post_bias, ("layer",), post)):
        if t is None:
            continue
        _check(t, name, x)
        if kind not in kinds:
            raise ValueError(f"{name}: the norm {kind!r} has none")
        if t.shape != (d,):
            raise RuntimeError(f"{name}: shape ({d},) expected, got {tuple(t.shape)}")
        if t.dtype != next(q for q in par if q is not None).dtype:
            raise RuntimeError("the norms' weights and biases share one dtype")
    rows = 0
    if gate is not None:
        _check(gate, "gate", x)
        rows = _gate_rows(gate, x)
    opt = (_NORMS[pre], _NORMS[post], float(scale), float(eps), float(p), _seed(seed, p), int(stream) & (2 ** 64 - 1), rows)
    if _wants_grad(x, f, gate, *par):
        return _ResidualNorm.apply(x, f, gate, *par, opt)
    y, h, _ = _res_forward(x, f, gate, *par, opt, False)
    return (x if y is None else y), h


# -- linear_cross_entropy -----------------------------------------------------------------------------------------------


def _lce_call(x, w, target, ignore, row_weight, reduction, want_x, want_w):
    """(losses, their mean or sum (reduction "none": None), dx, dw)"""
    (xr, ldx), (wr, ldw), t = _rows(x), _rows(w), target.contiguous()
    n, d = t.numel(), x.shape[-1]
    loss = torch.empty(n, device=x.device, dtype=torch.float32)
    total = None if reduction == "none" else torch.empty((), device=x.device, dtype=torch.float32)
    dx = x.new_empty(x.shape) if want_x else None
    dw = w.new_empty(w.shape) if want_w else None
    if not n:
        return loss, None if total is None else total.zero_(), dx, None if dw is None else dw.zero_()
    _run_ws(x, L.lib().psgdk_linear_cross_entropy, n, d, w.shape[0], L.dtype_code(x.dtype), xr.data_ptr(), ldx, wr.data_ptr(),
            ldw, t.data_ptr(), ignore, _ptr(row_weight), int(reduction == "mean"), loss.data_ptr(), _ptr(total), _ptr(dx), d,
            _ptr(dw), d)
    return loss, total, dx, dw


class _LinearCrossEntropy(torch.autograd.Function):
    """A reduced loss has its gradients ready in the forward pass (they cost one third less than with the logits computed
    again) and hands them over in the backward pass, scaled by the loss's gradient; where the graph is kept for another
    backward pass they are computed again. bfloat16 gradients are rounded a second time by that scaling: it costs them less
    than the float32 ones between the passes would take in memory (twice dx and dw) or a third set of products in time, and
    nothing where the scale is a power of two. The losses of single rows need their gradients' weights first."""

    @staticmethod
    def forward(ctx, x, w, target, ignore, reduction):
        reduced = reduction != "none"
        need = ctx.needs_input_grad
        loss, total, dx, dw = _lce_call(x, w, target, ignore, None, reduction, reduced and need[0], reduced and need[1])
        ctx.save_for_backward(x, w, target, dx, dw)  # all of them: hooks on saved tensors move or drop the gradients too
        ctx.args = ignore, reduction
        ctx.handed_over = False
        return total if reduced else loss.view(target.shape)

    @staticmethod
    def backward(ctx, g):
        _once()
        x, w, target, *grads = ctx.saved_tensors
        ignore, reduction = ctx.args
        need = ctx.needs_input_grad
        if reduction == "none":
            g = g.reshape(-1).float().contiguous()
            return (*_lce_call(x, w, target, ignore, g, reduction, need[0], need[1])[2:], None, None, None)
        if ctx.handed_over:
            grads = _lce_call(x, w, target, ignore, None, reduction, need[0], need[1])[2:]
        else:  # (.data: what the caller does to them in place is no change of a saved tensor)
            grads = [None if t is None else t.data for t in grads]
            ctx.handed_over = True
        ts = [t for t in grads if t is not None and t.numel()]
        if ts:
            g = g.float()
            n = (C.c_int64 * len(ts))(*[t.numel() for t in ts])
            _run(x, L.lib().psgdk_scale_by, len(ts), n, L.dtype_code(x.dtype), L.ptrs(ts), g.data_ptr())
        return (*grads, None, None, None)


def linear_cross_entropy(x, weight, target, *, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of the logits x weight^T, which are never kept: x (..., d), weight (vocabulary, d) in x's
    dtype, target (...) of int64. Rows whose target is ignore_index have no loss and no gradient, whatever x holds there;
    another target outside the vocabulary makes the loss NaN. reduction: "mean" over the rows not ignored (0 where there
    are none), "sum", or "none" (losses in target's shape). Losses are float32; the gradients of x and weight have their
    dtype. With bfloat16 they are sums over logits' gradients rounded to bfloat16 ("none": weighted and rounded), and where
    a mean or sum is scaled afterwards by other than a power of two they are rounded again; float32 keeps its bits."""
    _check(x, "x")
    _check(weight, "weight", x)
    if weight.dtype != x.dtype:
        raise RuntimeError(f"weight: {x.dtype} expected as x, got {weight.dtype}")
    if x.dim() == 0 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or not weight.numel():
        raise RuntimeError(f"x {tuple(x.shape)}, weight {tuple(weight.shape)}: (..., d) and (vocabulary, d) expected")
    if target.dtype != torch.int64 or target.device != x.device or target.shape != x.shape[:-1]:
        raise RuntimeError(f"target: int64 {tuple(x.shape[:-1])} on {x.device} expected, got {target.dtype} "
                           f"{tuple(target.shape)} on {target.device}")
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction = {reduction!r}: 'mean', 'sum' or 'none'")
    if _wants_grad(x, weight):
        return _LinearCrossEntropy.apply(x, weight, target, int(ignore_index), reduction)
    loss, total, _, _ = _lce_call(x, weight, target, int(ignore_index), None, reduction, False, False)
    return loss.view(target.shape) if reduction == "none" else total
