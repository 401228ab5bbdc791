"""How far linear_cross_entropy's losses and gradients are off, and that no part of the vocabulary or of the rows is left out,
on the GPU against float64.

The bounds of test_train_ops.py are for roundings that all go one way. Here errors are taken together: the error of one
rounding to bfloat16 is spread evenly over half a unit of the last place either way, 2^-8 / sqrt(3) of a value at 1 and half
of that at 2, in the mean square over a factor of two STEP = .00166. A coded logit is off by up to 2^-10, CODE = .00056 in
the mean square. Independent errors of a gradient's terms add up as their squares do."""
import math

import pytest
import torch

import psgd_pro_amd as P
from test_train_ops import DEV, DTYPES, E, rnd, run_lce, targets

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -8 / math.sqrt(3) * math.sqrt(3 / (8 * math.log(2)))
CODE = 2.0 ** -10 / math.sqrt(3)


@pytest.fixture(autouse=True)
def _lib(hip):
    return hip


# with gradients: up to 512 rows and 2^23 logits, many rows, rows and dx in parts; without: also a few rows
SIZES = [(300, 256, 1003), (400, 136, 16384), (700, 512, 4099), (1531, 770, 5021), (2048, 128, 32768)]


@pytest.mark.parametrize("scale", [1.0, 1.0 / 3.0])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,v", SIZES)
def test_gradients_are_as_near_as_their_roundings(dtype, n, d, v, scale):
    x, w, t = rnd((n, d), 1, dtype), rnd((v, d), 2, dtype, 1.5 / math.sqrt(d)), targets(n, v, 3, 0.2)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    gx, gw = torch.autograd.grad(P.linear_cross_entropy(xs, ws, t) * scale, (xs, ws))
    X, W, kept = x.double(), w.double(), t != -100
    dz = torch.softmax(X @ W.t(), 1)
    dz[torch.arange(n, device=DEV), t.clamp(min=0)] -= 1.0
    dz *= kept[:, None] * (scale / int(kept.sum()))
    for out, ref, terms in ((gx, dz @ W, dz.square() @ W.square()), (gw, dz.t() @ X, dz.square().t() @ X.square())):
        if dtype == torch.bfloat16:  # logits' gradients, stored gradient, and again after a scale that is no power of two
            var = (STEP ** 2 + CODE ** 2) * float(terms.sum()) + (1 + (scale != 1.0)) * STEP ** 2 * float(ref.square().sum())
        else:  # a logit's error (d roundings) times its softmax entry, sums of n or v terms, the stored gradient
            var = ((d + 64) + (n + v + 64) + 8) * E ** 2 * 4 * float(terms.sum()) + 2 * E ** 2 * float(ref.square().sum())
        assert float((out.double() - ref).norm()) <= 1.25 * math.sqrt(var), (float((out.double() - ref).norm() / ref.norm()),
                                                                             math.sqrt(var) / float(ref.norm()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v", [(16, 50048), (40, 16384), (300, 16384), (520, 16500), (1100, 32896)])
def test_no_part_of_the_vocabulary_is_left_out(dtype, n, v):
    """Each 128 entries of the vocabulary have a column of their own, which only they reach: a gradient's column is their
    share of the softmax alone."""
    d = (v + 127) // 128
    w = torch.zeros((v, d), device=DEV, dtype=dtype)
    w[torch.arange(v, device=DEV), torch.arange(v, device=DEV) // 128] = 1.0
    run_lce(rnd((n, d), 5, dtype, 0.5), w, targets(n, v, 6, 0.1), reductions=("mean",))
