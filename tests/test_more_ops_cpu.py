"""window_attention, qk_norm_rope and the AdamW step without a GPU: argument checks of the C ABI before any device work, workspace
sizes, the plan of a launch, and the Python entry points' refusals."""
import ctypes as C
import math

import pytest
import torch

import psgd_pro_amd as P
from psgd_pro_amd import _lib as L

PTR = 0x10000


def _err():
    return L.lib().psgdk_last_error().decode()


def heads(p=PTR, sb=4096, sn=256, sh=32):
    return L.Heads(p, sb, sn, sh)


def attn(**kw):
    a = L.WindowAttention(batch=2, n=16, m=16, heads=8, kv_heads=2, d=32, dtype=L.BF16, window=0, sinks=0, scale=0.1, q=heads(),
                          k=heads(sn=64), v=heads(sn=64), o=PTR, lse=PTR)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD_ATTN = [
    (dict(dtype=2), L.EINVAL), (dict(batch=0), L.ESHAPE), (dict(n=0), L.ESHAPE), (dict(m=0), L.ESHAPE), (dict(n=(1 << 28) + 1), L.ESHAPE),
    (dict(m=(1 << 28) + 1), L.ESHAPE), (dict(heads=0), L.ESHAPE), (dict(kv_heads=0), L.ESHAPE), (dict(kv_heads=3), L.ESHAPE), (dict(d=0), L.ESHAPE),
    (dict(d=136), L.ESHAPE), (dict(d=20), L.ESHAPE), (dict(window=-1), L.EINVAL), (dict(sinks=-1), L.EINVAL), (dict(scale=0.0), L.EINVAL),
    (dict(scale=-1.0), L.EINVAL), (dict(scale=math.nan), L.EINVAL), (dict(scale=math.inf), L.EINVAL),
    (dict(n=1 << 27, heads=32, kv_heads=1), L.ESHAPE), (dict(batch=1 << 20, n=1 << 12), L.ESHAPE)]
BAD_POINTERS = [
    (dict(q=heads(p=None)), L.EINVAL), (dict(k=heads(p=PTR + 8)), L.EINVAL), (dict(v=heads(sn=60)), L.ESHAPE), (dict(q=heads(sh=36)), L.ESHAPE),
    (dict(q=heads(sb=4100)), L.ESHAPE), (dict(k=heads(sb=-4096)), L.ESHAPE), (dict(k=heads(sn=-64)), L.ESHAPE), (dict(v=heads(sn=1 << 22)), L.ESHAPE),
    (dict(q=heads(sh=1 << 22)), L.ESHAPE), (dict(o=None), L.EINVAL), (dict(o=PTR + 2), L.EINVAL), (dict(o_rest=PTR + 8), L.EINVAL)]


@pytest.mark.parametrize("kw,code", BAD_ATTN + BAD_POINTERS)
def test_attention_refusals(kw, code):
    size = C.c_size_t(1 << 40)
    assert L.lib().psgdk_window_attention(C.byref(attn(**kw)), PTR, C.byref(size), None) == code, _err()
    assert _err()


@pytest.mark.parametrize("kw,code", BAD_ATTN + BAD_POINTERS + [(dict(lse=None), L.EINVAL), (dict(batch=1 << 20, m=1 << 12), L.ESHAPE)])
def test_attention_backward_refusals(kw, code):
    g, size = L.WindowAttentionGrads(heads(), PTR, PTR, PTR), C.c_size_t(1 << 40)
    assert L.lib().psgdk_window_attention_backward(C.byref(attn(**kw)), C.byref(g), PTR, C.byref(size), None) == code, _err()


def test_attention_gradient_blocks_and_workspaces():
    f, size = L.lib().psgdk_window_attention_backward, C.c_size_t(1 << 40)
    a, null = attn(), C.POINTER(L.WindowAttentionGrads)()
    assert f(C.byref(a), null, PTR, C.byref(size), None) == L.EINVAL
    assert f(None, null, PTR, C.byref(size), None) == L.EINVAL
    assert f(C.byref(a), C.byref(L.WindowAttentionGrads(heads(), PTR, PTR, PTR)), PTR, None, None) == L.EINVAL
    assert f(C.byref(a), C.byref(L.WindowAttentionGrads(heads(p=None), PTR, PTR, PTR)), PTR, C.byref(size), None) == L.EINVAL
    for grads in ((PTR + 4, PTR, PTR), (PTR, PTR + 8, PTR), (PTR, PTR, PTR + 2)):
        assert f(C.byref(a), C.byref(L.WindowAttentionGrads(heads(), *grads)), PTR, C.byref(size), None) == L.EINVAL and "alignment" in _err()
    # too small a workspace is refused
    assert f(C.byref(a), C.byref(L.WindowAttentionGrads(heads(), PTR, PTR, PTR)), None, C.byref(size), None) == L.OK
    need = size.value
    assert need >= 2 * 8 * 16 * 4
    size.value = need - 1
    assert f(C.byref(a), C.byref(L.WindowAttentionGrads(heads(), PTR, PTR, PTR)), PTR, C.byref(size), None) == L.EWORKSPACE


def query(fn, a, *more):
    size = C.c_size_t(0)
    assert fn(C.byref(a), *more, None, C.byref(size), None) == L.OK, _err()
    return size.value


def test_attention_workspaces_are_bounded():
    """Sums of parts are there only where there are few tiles, or first tokens that all rows see: up to 512 MiB, beside two numbers a row
    backward."""
    fwd, bwd = L.lib().psgdk_window_attention, L.lib().psgdk_window_attention_backward
    g = C.byref(L.WindowAttentionGrads(heads(), PTR, PTR, PTR))
    assert query(fwd, attn(n=4096, m=4096, batch=32, heads=32, kv_heads=8, d=128)) == 0
    token = query(fwd, attn(n=1, m=131072, batch=1, heads=32, kv_heads=8, d=128))
    assert 0 < token < 8 << 20
    assert query(fwd, attn(n=1, m=1 << 28, batch=1, heads=32, kv_heads=8, d=128)) < 8 << 20
    for kw in (dict(n=1, m=1 << 26, batch=1), dict(n=300, m=1 << 20, batch=2), dict(n=1 << 20, m=1 << 20, batch=8, window=100, sinks=1000)):
        a = attn(heads=32, kv_heads=8, d=128, **kw)
        assert query(fwd, a) < 200 << 20
        assert query(bwd, a, g) <= (512 << 20) + 256 * 4 + 8 * 32 * kw["n"] * kw["batch"]
    only_q = C.byref(L.WindowAttentionGrads(heads(), PTR, None, None))
    assert query(bwd, attn(n=4096, m=4096, window=50, sinks=4), only_q) == 2 * 4 * 2 * 8 * 4096


def rope(**kw):
    a = L.QkNormRope(batch=2, n=4, heads=4, kv_heads=2, d=32, rotary_dim=32, dtype=L.BF16, w_dtype=L.F32, norm=L.NORM_RMS, interleaved=0, eps=1e-6,
                     theta=1e4, q=heads(), k=heads(), q_w=PTR, k_w=PTR)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=5), L.EINVAL), (dict(w_dtype=5), L.EINVAL), (dict(batch=0), L.ESHAPE), (dict(n=0), L.ESHAPE), (dict(batch=1 << 20, n=1 << 20), L.ESHAPE),
    (dict(heads=0), L.ESHAPE), (dict(kv_heads=-1), L.ESHAPE), (dict(d=1), L.ESHAPE), (dict(d=33), L.ESHAPE), (dict(d=514), L.ESHAPE),
    (dict(rotary_dim=34), L.ESHAPE), (dict(rotary_dim=-2), L.ESHAPE), (dict(rotary_dim=3), L.ESHAPE), (dict(norm=3), L.EINVAL), (dict(eps=-1.0), L.EINVAL),
    (dict(eps=math.nan), L.EINVAL), (dict(theta=0.9), L.EINVAL), (dict(theta=math.inf), L.EINVAL), (dict(theta=math.nan), L.EINVAL),
    (dict(norm=L.NORM_NONE), L.EINVAL), (dict(q=heads(p=None)), L.EINVAL), (dict(k=heads(p=None)), L.EINVAL), (dict(kv_heads=0), L.EINVAL)])
def test_rope_refusals(kw, code):
    assert L.lib().psgdk_qk_norm_rope(C.byref(rope(**kw)), PTR, PTR, None) == code, _err()
    size = C.c_size_t(1 << 30)
    g = L.QkNormRopeGrads(heads(), heads(), PTR, PTR, PTR, PTR)
    assert L.lib().psgdk_qk_norm_rope_backward(C.byref(rope(**kw)), C.byref(g), PTR, C.byref(size), None) == code, _err()


def test_rope_outputs_and_workspace():
    f, b = L.lib().psgdk_qk_norm_rope, L.lib().psgdk_qk_norm_rope_backward
    assert f(C.byref(rope()), None, PTR, None) == L.EINVAL and f(C.byref(rope()), PTR, None, None) == L.EINVAL
    assert f(None, PTR, PTR, None) == L.EINVAL
    size = C.c_size_t(0)

    def back(a, *grads, ws=None):
        return b(C.byref(a), C.byref(L.QkNormRopeGrads(heads(), heads(), *grads)), ws, C.byref(size), None)

    assert back(rope(), PTR, PTR, None, None) == L.OK and size.value == 0
    assert back(rope(), None, None, None, None, ws=PTR) == L.OK  # nothing to do
    assert back(rope(), PTR, PTR, PTR, None) == L.OK and size.value == 2 * 1024 * 32 * 4
    size.value = 16
    assert back(rope(), PTR, PTR, PTR, PTR, ws=PTR) == L.EWORKSPACE
    assert back(rope(q_w=None), PTR, PTR, PTR, None) == L.EINVAL and back(rope(k_w=None), PTR, PTR, None, PTR) == L.EINVAL
    assert back(rope(kv_heads=0, k_w=None), PTR, PTR, None, None) == L.EINVAL
    assert b(C.byref(rope()), None, None, C.byref(size), None) == L.EINVAL
    assert b(C.byref(rope()), C.byref(L.QkNormRopeGrads()), None, None, None) == L.EINVAL


def adamw(sizes=(5, 300), bits=32, dtypes=None, **kw):
    n = len(sizes)
    keep = dict(n=(C.c_int64 * n)(*sizes), dtype=(C.c_int32 * n)(*(dtypes or [0] * n)), **{k: L.ptrs([PTR] * n) for k in ("p", "g", "m", "v", "m_scale", "v_scale")})
    a = L.AdamW(nb=n, bits=bits, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, step=1)
    for k, v in keep.items():
        setattr(a, k, C.cast(v, C.c_void_p))
    for k, v in kw.items():
        setattr(a, k, C.cast(v, C.c_void_p) if isinstance(v, C.Array) else v)
    a.keep = keep, kw
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(bits=16), L.EINVAL), (dict(nb=-1), L.ESHAPE), (dict(nb=(1 << 20) + 1), L.ESHAPE), (dict(lr=math.nan), L.EINVAL), (dict(weight_decay=math.inf), L.EINVAL),
    (dict(eps=-1.0), L.EINVAL), (dict(eps=math.nan), L.EINVAL), (dict(beta1=1.0), L.EINVAL), (dict(beta2=-0.1), L.EINVAL), (dict(beta1=math.nan), L.EINVAL),
    (dict(step=0), L.ESHAPE), (dict(step=(1 << 32) + 1), L.ESHAPE), (dict(max_norm=-1.0), L.EINVAL), (dict(max_norm=math.nan), L.EINVAL), (dict(n=None), L.EINVAL),
    (dict(dtype=None), L.EINVAL), (dict(g=None), L.EINVAL), (dict(m=None), L.EINVAL), (dict(v=None), L.EINVAL), (dict(bits=8, m_scale=None), L.EINVAL),
    (dict(bits=8, v_scale=None), L.EINVAL), (dict(dtypes=[0, 2]), L.EINVAL), (dict(sizes=(5, -1)), L.ESHAPE), (dict(sizes=(5, (1 << 40) + 1)), L.ESHAPE),
    (dict(p=L.ptrs([PTR, None])), L.EINVAL), (dict(g=L.ptrs([None, PTR])), L.EINVAL), (dict(v=L.ptrs([None, PTR])), L.EINVAL),
    (dict(bits=8, m_scale=L.ptrs([None, PTR])), L.EINVAL)])
def test_adamw_refusals(kw, code):
    size = C.c_size_t(1 << 30)
    assert L.lib().psgdk_adamw(C.byref(adamw(**kw)), PTR, C.byref(size), None) == code, _err()


def test_adamw_workspace():
    f = L.lib().psgdk_adamw
    assert f(None, None, None, None) == L.EINVAL and f(C.byref(adamw()), None, None, None) == L.EINVAL
    assert query(f, adamw()) == 0
    assert query(f, adamw(max_norm=1.0)) == 256 + 4  # two workgroups' sums, and the factor
    assert query(f, adamw(norm=PTR)) == 16
    assert query(f, adamw(sizes=(1 << 39, 7), max_norm=1.0)) < 8 << 20
    size = C.c_size_t(4)
    assert f(C.byref(adamw(max_norm=1.0)), PTR, C.byref(size), None) == L.EWORKSPACE
    assert f(C.byref(adamw(sizes=())), PTR, C.byref(size), None) == L.OK and f(C.byref(adamw(sizes=(0, 0))), PTR, C.byref(size), None) == L.OK


def test_python_entry_points_take_gpu_tensors_only():
    x = torch.zeros(1, 4, 2, 8)
    for call in (lambda: P.window_attention(x, x, x), lambda: P.qk_norm_rope(x, x), lambda: P.adamw_step([x], [x], [x], [x], step=1),
                 lambda: P.AdamW([x.clone().requires_grad_()])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_adamw_states():
    like = torch.zeros(3, 100)
    assert P.adamw_state(like).shape == like.shape and P.adamw_state(like).dtype == torch.float32
    codes, scales = P.adamw_state(like, 8)
    assert codes.shape == (300,) and codes.dtype == torch.float8_e4m3fn and scales.shape == (2,) and scales.dtype == torch.float8_e8m0fnu
    assert not codes.float().any()
    with pytest.raises(ValueError):
        P.adamw_state(like, 4)
