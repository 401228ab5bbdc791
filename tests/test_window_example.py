"""The operators in a run together, as examples/train_lm.py has them with a window: queries and keys normalised and rotated,
attention, residual sums and norms, the loss, and both optimizers' steps."""
import importlib.util
import math
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_lm.py")
    spec = importlib.util.spec_from_file_location("train_lm", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def rms(v, w):
    return v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w


def rotate(u):
    n, d = u.shape[1], u.shape[-1]
    t = torch.arange(n, device=DEV, dtype=torch.float64)[:, None, None] * 10000.0 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
    a, b = u[..., :d // 2], u[..., d // 2:]
    return torch.cat((a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()), -1)


def plain_loss(m, leaves, tokens, targets):
    """The model's loss without dropout in elementary operations on `leaves` (the model's parameters in float64)."""
    it = iter(leaves)
    embed, head = next(it), next(it)
    norms, gates = [next(it) for _ in m.norms], [next(it) for _ in m.gates]
    head_norms = [next(it) for _ in m.head_norms]
    batch, n = tokens.shape
    i, j = torch.arange(n, device=DEV)[:, None], torch.arange(n, device=DEV)
    see = (j <= i) & ((i - j < m.window) | (j < m.sinks))
    y = embed[tokens]
    h = rms(y, norms[0])
    for k in range(m.layers):
        qkv, proj, up, down = (next(it) for _ in range(4))
        q, key, v = (h @ qkv.t()).view(batch, n, m.heads + 2 * m.kv, -1).split((m.heads, m.kv, m.kv), 2)
        q, key = rotate(rms(q, head_norms[2 * k])), rotate(rms(key, head_norms[2 * k + 1]))
        key, v = (t.repeat_interleave(m.heads // m.kv, 2) for t in (key, v))
        s = (q.transpose(1, 2) @ key.permute(0, 2, 3, 1).contiguous()) / math.sqrt(q.shape[-1])
        a = torch.softmax(s.masked_fill(~see, -math.inf), -1) @ v.transpose(1, 2).contiguous()
        y = y + gates[2 * k] * (a.transpose(1, 2).flatten(2) @ proj.t())
        h = rms(y, norms[2 * k + 1])
        y = y + gates[2 * k + 1] * (torch.nn.functional.gelu(h @ up.t()) @ down.t())
        h = rms(y, norms[2 * k + 2])
    z = h @ head.t()
    keep = targets >= 0
    return -(torch.log_softmax(z, -1)[keep].gather(1, targets[keep][:, None])).mean()


def test_gradients_of_the_whole_step(example, hip):
    """float32, against float64 autograd. Some thirty operations in a row, of sums of up to 512 terms: each adds at most about
    its terms' rounding, 512 E = 3e-5, to a gradient's norm, in all below 2^-10; a missing or wrong term is far above."""
    gen = torch.Generator(device=DEV).manual_seed(3)
    m = example.Model(512, 256, 2, 4, torch.device(DEV), gen, window=20, sinks=3)
    tokens, targets = example.batch_of(3, 75, 512, torch.device(DEV), gen)
    with torch.no_grad():
        for w in (*m.norms, *m.gates, *m.head_norms):
            w += 0.1 * torch.randn(w.shape, generator=gen, device=DEV)
    loss = m.loss(tokens, targets, 0.0, seed=0, dtype=torch.float32)
    grads = torch.autograd.grad(loss, m.parameters())
    leaves = [p.detach().double().requires_grad_() for p in m.parameters()]
    want = plain_loss(m, leaves, tokens, targets)
    assert abs(float(loss) - float(want)) < 2 ** -10
    for k, (g, r) in enumerate(zip(grads, torch.autograd.grad(want, leaves))):
        assert float((g.double() - r).norm()) <= 2 ** -10 * float(r.norm()), k


def test_example_runs_with_a_window(example, hip):
    losses = example.train(steps=6, vocab=1024, batch=4, tokens=200, window=33, sinks=2, log=lambda *_: None)
    assert len(losses) == 6 and all(math.isfinite(v) for v in losses)
