"""The training operators' Python side without a GPU: the entry points on CPU tensors, their launches recorded instead of
made (outputs hold nothing)."""
import ctypes as C
import weakref

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import psgd_pro_amd as P
from psgd_pro_amd import _lib as L
from psgd_pro_amd import train as T


@pytest.fixture
def calls(monkeypatch):
    """(entry point's name, arguments) of each launch."""
    made = []
    monkeypatch.setattr(T, "_check", lambda *a, **k: None)
    for name in ("_run", "_run_ws"):
        monkeypatch.setattr(T, name, lambda t, fn, *args: made.append((fn.__name__, args)))
    return made


@pytest.fixture(params=[torch.float64, torch.bfloat16, torch.float16])
def default_dtype(request):
    before = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield request.param
    torch.set_default_dtype(before)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("grad", [False, True])
def test_losses_are_float32_under_any_default_dtype(calls, default_dtype, reduction, grad):
    """The library writes 4 bytes for each loss."""
    x, w = torch.ones(6, 8, dtype=torch.float32, requires_grad=grad), torch.ones(5, 8, dtype=torch.float32)
    out = P.linear_cross_entropy(x, w, torch.zeros(6, dtype=torch.int64), reduction=reduction)
    assert out.dtype == torch.float32 and len(calls) == 1
    assert T._lce_call(x.detach(), w, torch.zeros(6, dtype=torch.int64), -100, None, reduction, False, False)[0].dtype == torch.float32


def test_row_statistics_are_float32_under_any_default_dtype(calls, default_dtype):
    """The library writes 16 bytes for each row's statistics."""
    x = torch.ones(6, 8, dtype=torch.float32, requires_grad=True)
    y, h = P.residual_norm(x, x)
    assert y.dtype == h.dtype == torch.float32 and len(calls) == 1
    stats = y.grad_fn.saved_tensors[-1]
    assert stats.shape == (6, 4) and stats.dtype == torch.float32


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode_is_refused(calls, grad, no_grad):
    """A tangent would be lost without a word. It is refused whichever input carries it, also where no input requires grad,
    and the same call without tangents goes through inside a dual level."""
    x, w = torch.ones(4, 8), torch.ones(5, 8)
    v, t = torch.ones(8), torch.zeros(4, dtype=torch.int64)
    ops = {
        "dropout": (lambda x: P.dropout(x, 0.5, seed=1), (x,)),
        "residual_norm": (lambda x, f, pw, pb, qw, qb, g: P.residual_norm(
            x, f, pre="layer", post="layer", pre_weight=pw, pre_bias=pb, post_weight=qw, post_bias=qb, gate=g),
            (x, x.clone(), v, v.clone(), v.clone(), v.clone(), v.clone())),
        "linear_cross_entropy": (lambda x, w: P.linear_cross_entropy(x, w, t), (x, w)),
    }
    with fwAD.dual_level(), torch.set_grad_enabled(not no_grad):
        for name, (op, args) in ops.items():
            args = [a.clone().requires_grad_(grad) for a in args]
            for k, a in enumerate(args):
                dual = fwAD.make_dual(a, torch.ones_like(a))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    op(*args[:k], dual, *args[k + 1:])
            assert not calls, name
            op(*args)
            assert len(calls) == 1, name
            calls.clear()


def test_forward_mode_transform_is_refused(calls):
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda x: P.dropout(x, 0.5, seed=1), (torch.ones(4, 8),), (torch.ones(4, 8),))
    assert not calls


@pytest.mark.parametrize("need", [(True, True), (True, False), (False, True)])
def test_gradients_made_ahead_are_saved_tensors(calls, need):
    """Hooks that move saved tensors away or drop them get the gradients that a reduced loss made in its forward pass, and
    nothing else keeps them."""
    x, w = (torch.ones(n, 8).requires_grad_(q) for n, q in zip((4, 5), need))
    t, held = torch.zeros(4, dtype=torch.int64), []

    def pack(q):
        held.append((q.shape, weakref.ref(q.untyped_storage())))
        return q.shape, q.dtype

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda q: torch.full(q[0], 7, dtype=q[1])):
        out = P.linear_cross_entropy(x, w, t)
    made = [shape for shape, storage in held if storage() is None]  # (x, w and the targets are still here)
    wanted = [q for q in (x, w) if q.requires_grad]
    assert made == [q.shape for q in wanted]
    for g, q in zip(torch.autograd.grad(out, wanted), wanted):
        assert torch.equal(g, torch.full_like(q, 7))
    assert [c[0] for c in calls] == ["psgdk_linear_cross_entropy", "psgdk_scale_by"]


def test_a_second_backward_pass_makes_the_gradients_again(calls):
    x = torch.ones(4, 8, requires_grad=True)
    out = P.linear_cross_entropy(x, torch.ones(5, 8), torch.zeros(4, dtype=torch.int64))
    a, = torch.autograd.grad(out, x, retain_graph=True)
    a.mul_(2)  # the caller's to change
    b, = torch.autograd.grad(out, x)
    assert a.data_ptr() != b.data_ptr()
    assert [c[0] for c in calls] == ["psgdk_linear_cross_entropy", "psgdk_scale_by"] * 2


@pytest.mark.parametrize("rows,d,vocab", [(500000, 4096, 1000), (1 << 20, 1024, 16), (4096, 4096, 131072), (1531, 770, 50021),
                                          (512, 1024, 16384), (65536, 256, 1024), (1 << 25, 1, 2), (3, 16, 1 << 22)])
@pytest.mark.parametrize("dtype", [L.F32, L.BF16])
@pytest.mark.parametrize("grad", [False, True])
def test_cross_entropy_workspace_is_what_the_header_says(rows, d, vocab, dtype, grad):
    """A slab's logits and its copy of x, a copy of an unaligned head, parts of the gradients."""
    size, ptr = C.c_size_t(0), 0x10000
    out = ptr if grad else None
    assert L.lib().psgdk_linear_cross_entropy(rows, d, vocab, dtype, ptr, d, ptr, d, ptr, -100, None, 1, ptr, None, out, d, out, d,
                                              None, C.byref(size), None) == L.OK
    e, ld, up = (2, -(-d // 8) * 8, -(-vocab // 64) * 64) if dtype == L.BF16 else (4, d, -(-vocab // 4) * 4)
    slab = min(rows, max(256 if dtype == L.BF16 else 1, (1 << 30) // (up * e)), 1 << (23 if dtype == L.BF16 else 22))
    small = dtype == L.BF16 and rows <= 512 and rows * vocab <= 1 << 23
    logits = slab * up * (e + 4 * small) if grad or small or dtype == L.F32 else 0
    parts = 32 * min(slab, 4096) * ld * 4 + 32 * vocab * ld * 4 if grad else 0
    copies = slab * ld * e + (vocab * ld * e if dtype == L.BF16 and d % 8 else 0)
    each = rows * 4 + slab * 64 + slab * -(-vocab // 256) * 8 + (1 << 20)  # the order, what a row keeps, sums of 128 columns
    assert size.value <= logits + copies + parts + each
