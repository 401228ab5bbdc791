"""The AdamW step where gradients' squares leave float32, the clip over tensors of several launches, and what the 8-bit states'
rounding does in the long run."""
import math

import numpy as np
import pytest
import torch

import psgd_pro_amd as P
from test_adamw import DEV, DTYPES, E, U, formula, host, rnd, unpack, within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(hip):
    return hip


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("big", [2.0 ** 64, 1e25, 2.0 ** 125])
@pytest.mark.parametrize("max_norm", [None, 3e38])
def test_8_bits_take_gradients_whose_squares_overflow(dtype, big, max_norm):
    """Three steps with such a block, one such element in a block and an ordinary block. Moments are within a code's step of the
    formula's (an eighth of a value, or of the least code: 2^-9 of the scale), the parameter's change within what a moment off by
    an eighth, and its root, leave of it."""
    n = 768
    p, g = torch.ones(n, device=DEV, dtype=dtype), rnd((n,), 1, dtype)
    g[:256] *= big / 8
    g[300] = -big
    p, g = [p], [g]
    ms, vs = [P.adamw_state(p[0], 8)], [P.adamw_state(p[0], 8)]
    for step in (1, 2, 3):
        old = [torch.from_numpy(unpack(host(s[0]), host(s[1]))).to(DEV) for s in (ms[0], vs[0])]
        before = p[0].clone()
        P.adamw_step(p, g, ms, vs, step=step, seed=3, max_norm=max_norm)
        refs, bounds = formula(before, g[0], old[0], old[1] ** 2, step)
        # (formula's bounds end with the square's: the root made from a 2^-64th of its terms has four roundings more)
        within(p[0], refs[0], bounds[0] + 8 * E * (before.double() - refs[0]).abs(), step)
        for state, want in ((ms[0], refs[1]), (vs[0], refs[2].sqrt())):
            got = torch.from_numpy(unpack(host(state[0]), host(state[1]))).to(DEV)
            least = state[1].float().double().repeat_interleave(256) * 2.0 ** -9
            within(got, want, torch.maximum(want.abs() / 8, least) * (1 + 64 * E))


def test_32_bits_leave_an_element_whose_square_overflows():
    p, g = [torch.ones(600, device=DEV)], [rnd((600,), 1)]
    g[0][70] = 1e25
    alone = [t.clone() for t in (p[0], g[0])]
    alone[1][70] = 0.0
    ms, vs = ([P.adamw_state(p[0])] for _ in range(2))
    mz, vz = ([P.adamw_state(p[0])] for _ in range(2))
    for step in (1, 2):
        P.adamw_step(p, g, ms, vs, step=step, weight_decay=0.0)
        P.adamw_step(alone[:1], alone[1:], mz, vz, step=step, weight_decay=0.0)
        assert torch.equal(p[0], alone[0]) and float(p[0][70]) == 1.0
