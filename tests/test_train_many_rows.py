"""residual_norm's gradients where a workgroup of the backward pass takes several rows, at every kind of row: many more rows
than there are workgroups at once, in numbers that no chunk of rows divides. References in float64, bounds as in
test_train_ops.py."""
import pytest
import torch

from test_train_ops import DTYPES, run_res

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _lib(hip):
    return hip


def rows_of(d):
    """(long sequences, short ones): the backward pass has up to 1024 workgroups, 256 of them from 4096 columns on where
    rows stay in registers."""
    if d < 8 or d > 8192:
        return (2, 1051), (701, 3)
    return ((2, 1501), (1037, 3)) if d <= 4096 else ((2, 529), (521, 2))


CASES = [("rms", None), ("rms", "rms"), ("layer", None), ("layer", "layer")]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pre,post", CASES)
@pytest.mark.parametrize("gate", [None, "channel", "long sequence", "short sequence", "token"])
@pytest.mark.parametrize("d", [5, 264, 770, 1100, 2048, 2304, 4096, 4101, 8192, 8200])
def test_residual_norm_of_many_rows(dtype, pre, post, gate, d):
    long, short = rows_of(d)
    batch, tokens = short if gate == "short sequence" else long
    shape = {None: None, "channel": (d,), "token": (batch, tokens, d)}.get(gate, (batch, 1, d))
    run_res((batch, tokens, d), dtype, pre, post, shape, p=0.1 if d % 2 else 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("use", [("dy",), ("dh",)])
@pytest.mark.parametrize("d", [5, 520, 2304, 6000, 8200])
def test_residual_norm_of_many_rows_with_one_gradient_only(dtype, use, d):
    batch, tokens = rows_of(d)[1]
    run_res((batch, tokens, d), dtype, "rms", "rms" if d != 6000 else None, (batch, 1, d), use=use)
