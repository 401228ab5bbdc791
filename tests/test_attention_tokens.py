"""window_attention of few rows in bfloat16: its outputs are the exact ones rounded."""
import pytest
import torch

import psgd_pro_amd as P
from test_attention import DEV, inputs, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(hip):
    return hip


@pytest.mark.parametrize("b,n,m,h,kv,d,window,sinks", [
    (8, 1, 4000, 32, 8, 128, None, 0), (1, 1, 60000, 32, 8, 128, None, 0), (6, 2, 900, 16, 2, 64, 300, 4), (4, 16, 700, 8, 2, 96, None, 0),
    (32, 1, 200, 12, 4, 40, None, 0), (3, 64, 64, 4, 4, 128, None, 0), (2, 9, 5000, 6, 1, 32, 1000, 1)])
def test_few_rows_round_once(b, n, m, h, kv, d, window, sinks):
    """The kernel's own error is some 2^-18 of an output's norm (probabilities in 16 bits or more), a step of bfloat16 2^-8 of the
    value: the share of outputs whose exact value lies so near a border, small ones among them, is below a hundredth. Probabilities
    rounded to bfloat16 give a third of the outputs another value."""
    q, k, v, _ = inputs(b, n, m, h, kv, d, torch.bfloat16)
    lengths = torch.randint(n, m + 1, (b,), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    kw = dict(window=window, sinks=sinks, lengths=lengths, starts=lengths - n)
    want = reference(q, k, v, None, **kw)[0][0].to(torch.bfloat16)
    out = P.window_attention(q, k, v, **kw)
    off = (out != want).double().mean()
    assert float(off) < 0.01, float(off)
    assert bool(((out.double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs() + 2.0 ** -14 * want.double().norm() / want.numel() ** 0.5).all())
