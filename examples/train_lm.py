"""A small language model trained with the package alone: KronWhiten for the step, linear_cross_entropy for the head,
residual_norm between the blocks and dropout on the embeddings (attention and the products are torch's).

    python examples/train_lm.py [--steps 60] [--dim 256] [--layers 2] [--vocab 4096] [--batch 16] [--tokens 128] [--p 0.1]

The text is made up: each sequence counts upwards in a stride of its own, so that the next token follows from the last
two. Prints the loss every ten steps and one JSON line at the end. Parameters are float32, the forward pass bfloat16."""
import argparse
import json
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from psgd_pro_amd import KronWhiten, dropout, linear_cross_entropy, residual_norm  # noqa: E402


class Model:
    """Decoder of `layers` blocks with a norm before each half (attention, MLP) and a learned scale for each channel on
    what it adds to the residual stream."""

    def __init__(self, vocab, dim, layers, heads, dev, gen):
        def weight(rows, cols, gain=1.0):
            w = torch.randn(rows, cols, device=dev, generator=gen) * (gain / math.sqrt(cols))
            return w.requires_grad_()

        def ones(value=1.0):
            return torch.full((dim,), value, device=dev).requires_grad_()

        self.heads, self.layers = heads, layers
        self.embed = weight(vocab, dim, math.sqrt(dim))
        self.head = weight(vocab, dim)
        self.norms = [ones() for _ in range(2 * layers + 1)]
        self.gates = [ones(0.5) for _ in range(2 * layers)]
        self.blocks = [dict(qkv=weight(3 * dim, dim), proj=weight(dim, dim), up=weight(2 * dim, dim), down=weight(dim, 2 * dim))
                       for _ in range(layers)]

    def parameters(self):
        return [self.embed, self.head, *self.norms, *self.gates, *(w for b in self.blocks for w in b.values())]

    def loss(self, tokens, targets, p, seed):
        """Mean cross entropy; p, seed: the step's dropout, each call with a stream of its own."""
        batch, n = tokens.shape
        bf = torch.bfloat16
        x = dropout(self.embed.to(bf)[tokens], p, seed=seed)
        y, h = residual_norm(x, pre_weight=self.norms[0])
        for i, b in enumerate(self.blocks):
            q, k, v = (h @ b["qkv"].to(bf).t()).view(batch, n, 3, self.heads, -1).permute(2, 0, 3, 1, 4)
            a = torch.nn.functional.scaled_dot_product_attention(q, k, v, is_causal=True)
            a = a.transpose(1, 2).reshape(batch, n, -1) @ b["proj"].to(bf).t()
            y, h = residual_norm(y, a, pre_weight=self.norms[2 * i + 1], gate=self.gates[2 * i], p=p, seed=seed, stream=2 * i + 1)
            m = torch.nn.functional.gelu(h @ b["up"].to(bf).t()) @ b["down"].to(bf).t()
            y, h = residual_norm(y, m, pre_weight=self.norms[2 * i + 2], gate=self.gates[2 * i + 1], p=p, seed=seed,
                                 stream=2 * i + 2)
        return linear_cross_entropy(h, self.head.to(bf), targets)


def batch_of(batch, tokens, vocab, dev, gen):
    start = torch.randint(vocab, (batch, 1), device=dev, generator=gen)
    stride = torch.randint(1, 8, (batch, 1), device=dev, generator=gen)
    s = (start + stride * torch.arange(tokens + 1, device=dev)) % vocab
    targets = s[:, 1:].clone()
    targets[:, 0] = -100  # one token does not say the stride
    return s[:, :-1], targets


def train(steps=60, dim=256, layers=2, vocab=4096, batch=16, tokens=128, p=0.1, lr=3e-3, seed=0, log=print):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(seed)
    model = Model(vocab, dim, layers, dim // 64, dev, gen)
    opt = KronWhiten(model.parameters(), preconditioner_max_skew=2, momentum=0.9, lr_params=lr, precision="bf16", seed=seed)
    losses = []
    for step in range(steps):
        x, t = batch_of(batch, tokens, vocab, dev, gen)
        losses.append(opt.step(lambda: model.loss(x, t, p, seed=step)).detach().item())
        if step % 10 == 0:
            log(f"step {step:4d}  loss {losses[-1]:.4f}")
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    for name, value in (("steps", 60), ("dim", 256), ("layers", 2), ("vocab", 4096), ("batch", 16), ("tokens", 128)):
        ap.add_argument("--" + name, type=int, default=value)
    ap.add_argument("--p", type=float, default=0.1)
    a = ap.parse_args()
    out = train(**vars(a))
    print(json.dumps({"loss_first_last": [round(out[0], 4), round(sum(out[-5:]) / min(5, len(out)), 4)], **vars(a)}))
