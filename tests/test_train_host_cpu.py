"""The training operators' Python side without a GPU: the entry points on CPU tensors, their launches recorded instead of
made (outputs hold nothing)."""
import pytest
import torch

import psgd_pro_amd as P
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
