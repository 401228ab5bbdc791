"""qk_norm_rope where heads do not fill a wave and eps is 0, and its angles at far positions against extended precision."""
import pytest
import torch

from test_qk_norm_rope import DTYPES, check, rnd

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
