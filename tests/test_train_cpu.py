"""The training operators without a GPU: argument checks of the C ABI before any device work, workspace sizes, and the
Python entry points' refusals."""
import ctypes as C

import pytest
import torch

import psgd_pro_amd as P
from psgd_pro_amd import _lib as L

PTR = 0x10000


def _err():
    return L.lib().psgdk_last_error().decode()


def _res(**kw):
    a = L.ResidualNorm(rows=4, d=16, dtype=L.BF16, pre=L.NORM_RMS, post=L.NORM_RMS, eps=1e-6, scale=1.0, x=PTR, ldx=16,
                       f=PTR, ldf=16, y=PTR, ldy=16, h=PTR, ldh=16, stats=PTR)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_dropout_refusals():
    f = L.lib().psgdk_dropout
    ok = [4, 16, 1, PTR, 16, PTR, 16, 0.1, 0, 0, None]

    def with_(i, v):
        a = list(ok)
        a[i] = v
        return f(*a)

    assert with_(2, 2) == L.EINVAL and "dtype" in _err()
    assert with_(0, -1) == L.ESHAPE and "rows" in _err()
    assert with_(1, 0) == L.ESHAPE
    assert with_(3, None) == L.EINVAL and "x" in _err()
    assert with_(4, 15) == L.ESHAPE and "row stride" in _err()
    assert with_(5, None) == L.EINVAL
    assert with_(6, 8) == L.ESHAPE
    for p in (-0.1, 1.5, float("nan")):
        assert with_(7, p) == L.EINVAL and "p =" in _err()
    assert with_(0, 0) == L.OK  # nothing to do: no device work


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), L.EINVAL), (dict(d=0), L.ESHAPE), (dict(d=(1 << 20) + 1), L.ESHAPE), (dict(rows=-1), L.ESHAPE),
    (dict(rows=1 << 30), L.ESHAPE), (dict(pre=3), L.EINVAL), (dict(post=-1), L.EINVAL), (dict(eps=-1.0), L.EINVAL),
    (dict(eps=float("nan")), L.EINVAL), (dict(pre_b=PTR), L.EINVAL), (dict(post_b=PTR), L.EINVAL),
    (dict(pre=L.NORM_NONE, pre_w=PTR), L.EINVAL), (dict(post=L.NORM_NONE, post_w=PTR), L.EINVAL),
    (dict(f=None), L.EINVAL), (dict(f=None, post=L.NORM_NONE, p=0.5), L.EINVAL),
    (dict(f=None, post=L.NORM_NONE, gate_rows=1, gate=PTR, ldgate=16), L.EINVAL), (dict(pre_w=PTR, w_dtype=7), L.EINVAL),
    (dict(gate_rows=3, gate=PTR, ldgate=16), L.ESHAPE), (dict(gate_rows=2, gate=None, ldgate=16), L.EINVAL),
    (dict(gate_rows=2, gate=PTR, ldgate=8), L.ESHAPE), (dict(gate_rows=2, gate=PTR, ldgate=16, gate_dtype=9), L.EINVAL),
    (dict(p=2.0), L.EINVAL), (dict(ldf=8), L.ESHAPE), (dict(ldx=8), L.ESHAPE), (dict(x=None), L.EINVAL),
    (dict(ldy=8), L.ESHAPE), (dict(h=None), L.EINVAL), (dict(pre=L.NORM_NONE, y=None), L.EINVAL),
    (dict(stats=PTR + 4), L.EINVAL)])
def test_residual_norm_refusals(kw, code):
    assert L.lib().psgdk_residual_norm(C.byref(_res(**kw)), None) == code, _err()
    assert _err()


def test_residual_norm_backward_refusals_and_workspace():
    f = L.lib().psgdk_residual_norm_backward
    a = _res(rows=4096, gate_rows=8, gate=PTR, ldgate=16, gate_dtype=0)
    sz = C.c_size_t(0)

    def call(a, ws=None, size=None, **g):
        s = C.c_size_t(size or 0)
        rc = f(C.byref(a), C.byref(L.ResidualNormGrads(**g)), ws, C.byref(s), None)
        sz.value = s.value
        return rc

    assert f(C.byref(a), None, None, C.byref(sz), None) == L.EINVAL
    assert f(C.byref(a), C.byref(L.ResidualNormGrads()), None, None, None) == L.EINVAL
    assert call(a, dy=PTR, lddy=16, dx=PTR, lddx=16) == L.OK and sz.value == 0
    assert call(a, dh=PTR, lddh=16, dpre_w=PTR) == L.OK
    one = sz.value
    assert 0 < one <= 1024 * 16 * 4 + 256
    assert call(a, dh=PTR, lddh=16, dpre_w=PTR, dpost_w=PTR, dgate=PTR, lddgate=16) == L.OK and sz.value > 2 * one
    assert call(a, ws=PTR, size=16, dh=PTR, lddh=16, dpre_w=PTR) == L.EWORKSPACE
    assert call(_res(pre=L.NORM_NONE), dh=PTR, lddh=16) == L.EINVAL
    assert call(_res(pre=L.NORM_NONE), dpre_w=PTR) == L.EINVAL
    assert call(_res(post=L.NORM_NONE), dpost_w=PTR) == L.EINVAL
    assert call(_res(f=None, post=L.NORM_NONE), df=PTR, lddf=16) == L.EINVAL
    assert call(_res(), dgate=PTR, lddgate=16) == L.EINVAL
    assert call(_res(stats=None), ws=PTR, size=1 << 20, dh=PTR, lddh=16, dx=PTR, lddx=16) == L.EINVAL and "stats" in _err()
    assert call(_res(), ws=PTR, size=1 << 20, dh=PTR, lddh=8, dx=PTR, lddx=16) == L.ESHAPE


def test_cross_entropy_refusals_and_workspace():
    f = L.lib().psgdk_linear_cross_entropy
    sz = C.c_size_t(0)
    ok = dict(rows=64, d=32, vocab=1000, dtype=1, x=PTR, ldx=32, w=PTR, ldw=32, target=PTR, ignore=-100, rw=None, mean=1,
              loss=PTR, total=None, dx=PTR, lddx=32, dw=PTR, lddw=32, ws=None, sz=C.byref(sz), st=None)

    def call(**kw):
        return f(*{**ok, **kw}.values())

    assert call() == L.OK and sz.value > 0
    need = sz.value
    assert call(dx=None, dw=None) == L.OK and sz.value <= need
    assert call(dtype=4) == L.EINVAL
    assert call(rows=0) == L.ESHAPE and call(d=0) == L.ESHAPE and call(vocab=0) == L.ESHAPE
    assert call(sz=None) == L.EINVAL
    assert call(rw=PTR) == L.EINVAL and "exclude" in _err()
    sz.value = 16
    assert call(ws=PTR) == L.EWORKSPACE
    sz.value = need
    for name in ("x", "w", "target", "loss"):
        assert call(ws=PTR, **{name: None}) == L.EINVAL, name
    for name in ("ldx", "ldw", "lddx", "lddw"):
        assert call(ws=PTR, **{name: 31}) == L.ESHAPE, name
    # the logits never take more than a bounded part of memory, whatever the number of rows
    assert call(rows=1 << 20, vocab=1 << 17) == L.OK and sz.value < (3 << 30)


def test_scale_refusals():
    f = L.lib().psgdk_scale_by
    n = (C.c_int64 * 1)(4)
    assert f(0, n, 0, L.ptrs([PTR]), PTR, None) == L.EINVAL
    assert f(5, n, 0, L.ptrs([PTR]), PTR, None) == L.EINVAL
    assert f(1, n, 2, L.ptrs([PTR]), PTR, None) == L.EINVAL
    assert f(1, n, 0, L.ptrs([None]), PTR, None) == L.EINVAL
    assert f(1, n, 0, L.ptrs([PTR]), None, None) == L.EINVAL


def test_python_entry_points_take_gpu_tensors_only():
    x = torch.zeros(4, 8)
    for call in (lambda: P.dropout(x, 0.1), lambda: P.residual_norm(x, x),
                 lambda: P.linear_cross_entropy(x, x, torch.zeros(4, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
