"""examples/train_lm.py: the training operators and KronWhiten together."""
import importlib.util
import math
import os

import pytest

pytestmark = pytest.mark.gpu


def test_language_model_example_learns(hip):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_lm.py")
    spec = importlib.util.spec_from_file_location("train_lm", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses = mod.train(steps=40, log=lambda *_: None)
    # an untrained head is near the uniform distribution's log(vocab) plus half the variance of its logits (one)
    assert abs(losses[0] - (math.log(4096) + 0.5)) < 0.5
    assert all(math.isfinite(v) for v in losses)
    assert sum(losses[-5:]) / 5 < losses[0] - 1.0
