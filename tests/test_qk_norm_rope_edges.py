"""qk_norm_rope where heads do not fill a wave and eps is 0, and its angles at far positions against extended precision."""
import math
from decimal import Decimal, localcontext

import pytest
import torch

import psgd_pro_amd as P
from test_qk_norm_rope import DTYPES, E, check, rnd, within

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(hip):
    return hip


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("eps", [0.0, 1e-50])
@pytest.mark.parametrize("h,kv,d,rot", [(9, 3, 80, 80), (5, 1, 64, 32), (3, 1, 128, 128), (7, 2, 40, 20), (3, 5, 6, 4), (1, 1, 2, 2)])
def test_eps_of_zero_with_heads_that_leave_lanes_without_one(dtype, norm, eps, h, kv, d, rot):
    """Gradients of rows that are not zero are finite without eps (1e-50 is 0 in float32). Heads of 2 and 6 have few values: theirs
    are far enough apart that no row's deviation is near zero."""
    q, k = rnd((2, 11, h, d), 1, dtype, mean=0.3), rnd((2, 11, kv, d), 2, dtype, std=3.0)
    if d < 8:
        ramp = torch.arange(d, device=q.device, dtype=dtype) * 8
        q, k = q + ramp, k + 2 * ramp
    check(q, k, rnd((d,), 3, std=0.3, mean=1.0), rnd((d,), 4, std=0.3, mean=1.0), norm=norm, eps=eps, rotary_dim=rot)


PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def turned(x, positions, theta, interleaved):
    """x (n, heads, d) rotated, in float64 from angles reduced in 60 digits, and the pairs' partners."""
    half = x.shape[-1] // 2
    with localcontext() as ctx:
        ctx.prec = 60
        rates = [(Decimal(-i) / half * Decimal(theta).ln()).exp() / (2 * PI) for i in range(half)]
        turns = [[float(p * r - (p * r).to_integral_value()) for r in rates] for p in positions]
    t = 2 * math.pi * torch.tensor(turns, dtype=torch.float64, device=x.device)[:, None]
    x = x.double()
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    join = (lambda u, v: torch.stack((u, v), -1).flatten(-2)) if interleaved else (lambda u, v: torch.cat((u, v), -1))
    return join(a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()), join(b, a)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d", [64, 72, 512, 6])
@pytest.mark.parametrize("theta", [10000.0, 1.5, 1.01, 1e6])
def test_far_angles_against_extended_precision(theta, d, interleaved):
    """Within p 2^-48 of the definition's angle, beside the rotation's own rounding (8 E of the pair): forward at far positions,
    and the gradient, which is the rotation back."""
    positions = [3, (1 << 24) - 1, (1 << 24) + 5, (1 << 28) + 77, (1 << 31) - 1, -(1 << 31) - 9, -(1 << 34) + 1, (1 << 40) + 12345]
    pos = torch.tensor(positions, device="cuda:0")
    x, g = rnd((1, len(positions), 3, d), 1), rnd((1, len(positions), 3, d), 2)
    leaf = x.clone().requires_grad_()
    y, _ = P.qk_norm_rope(leaf, norm=None, positions=pos, theta=theta, interleaved=interleaved)
    for out, v, at in ((y, x, positions), (torch.autograd.grad(y, leaf, g)[0], g, [-p for p in positions])):
        want, partner = turned(v[0], at, theta, interleaved)
        angle = pos.double().abs()[:, None, None] * 2.0 ** -48
        within(out[0], want, (8 * E + angle) * (v[0].double().abs() + partner.abs()), theta)
