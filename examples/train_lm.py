"""A small language model trained with the package: KronWhiten for the step, linear_cross_entropy for the head, residual_norm
between the blocks and dropout on the embeddings (attention and the products are torch's). With --window the attention is the
package's too, and AdamW takes what is no matrix of a block: qk_norm_rope on grouped queries and keys, window_attention over
that many tokens and the first ones (--sinks), embeddings, norms and gates with states of 8 bits.

    python examples/train_lm.py [--steps 60] [--dim 256] [--layers 2] [--vocab 4096] [--batch 16] [--tokens 128] [--p 0.1]
                                [--window 32] [--sinks 2]

The text is made up: each sequence counts upwards in a stride of its own, so that the next token follows from the last
two. Prints the loss every ten steps and one JSON line at the end. Parameters are float32, the forward pass bfloat16."""
import argparse
import json
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from psgd_pro_amd import (AdamW, KronWhiten, dropout, linear_cross_entropy, qk_norm_rope, residual_norm,  # noqa: E402
                          window_attention)


class Model:
    """Decoder of `layers` blocks with a norm before each half (attention, MLP) and a learned scale for each channel on
    what it adds to the residual stream."""

    def __init__(self, vocab, dim, layers, heads, dev, gen, window=None, sinks=0):
        def weight(rows, cols, gain=1.0):
            w = torch.randn(rows, cols, device=dev, generator=gen) * (gain / math.sqrt(cols))
            return w.requires_grad_()

        def ones(value=1.0):
            return torch.full((dim,), value, device=dev).requires_grad_()

        self.heads, self.layers, self.window, self.sinks = heads, layers, window, sinks
        self.kv = heads if window is None else max(1, heads // 2)  # (with a window two query heads share a key head)
        rows = dim // heads * (heads + 2 * self.kv)
        self.embed = weight(vocab, dim, math.sqrt(dim))
        self.head = weight(vocab, dim)
        self.norms = [ones() for _ in range(2 * layers + 1)]
        self.gates = [ones(0.5) for _ in range(2 * layers)]
        self.blocks = [dict(qkv=weight(rows, dim), proj=weight(dim, dim), up=weight(2 * dim, dim), down=weight(dim, 2 * dim))
                       for _ in range(layers)]

        self.head_norms = [] if window is None else [torch.ones(dim // heads, device=dev).requires_grad_() for _ in range(2 * layers)]

    def matrices(self):
        return [w for b in self.blocks for w in b.values()]

    def others(self):
        return [self.embed, self.head, *self.norms, *self.gates, *self.head_norms]

    def parameters(self):
        return self.others() + self.matrices()

    def attention(self, i, qkv):
        """The heads' outputs (batch, n, dim) of layer i from its projection (batch, n, rows)."""
        batch, n, _ = qkv.shape
        if self.window is None:
            q, k, v = qkv.view(batch, n, 3, self.heads, -1).permute(2, 0, 3, 1, 4)
            return torch.nn.functional.scaled_dot_product_attention(q, k, v, is_causal=True).transpose(1, 2).reshape(batch, n, -1)
        q, k, v = qkv.view(batch, n, self.heads + 2 * self.kv, -1).split((self.heads, self.kv, self.kv), 2)
        q, k = qk_norm_rope(q, k, q_weight=self.head_norms[2 * i], k_weight=self.head_norms[2 * i + 1])
        return window_attention(q, k, v, window=self.window, sinks=self.sinks).flatten(2)

    def loss(self, tokens, targets, p, seed, dtype=torch.bfloat16):
        """Mean cross entropy; p, seed: the step's dropout, each call with a stream of its own."""
        bf = dtype
        x = dropout(self.embed.to(bf)[tokens], p, seed=seed)
        y, h = residual_norm(x, pre_weight=self.norms[0])
        for i, b in enumerate(self.blocks):
            a = self.attention(i, h @ b["qkv"].to(bf).t()) @ b["proj"].to(bf).t()
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


def train(steps=60, dim=256, layers=2, vocab=4096, batch=16, tokens=128, p=0.1, lr=3e-3, seed=0, window=None, sinks=0, log=print):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(seed)
    model = Model(vocab, dim, layers, dim // 64, dev, gen, window, sinks)
    whiten = model.parameters() if window is None else model.matrices()
    opt = KronWhiten(whiten, preconditioner_max_skew=2, momentum=0.9, lr_params=lr, precision="bf16", seed=seed)
    rest = None if window is None else AdamW(model.others(), lr_params=lr, max_norm=1.0, state_bits=8, seed=seed)
    losses = []
    for step in range(steps):
        x, t = batch_of(batch, tokens, vocab, dev, gen)
        if rest is None:
            losses.append(opt.step(lambda: model.loss(x, t, p, seed=step)).detach().item())
        else:
            loss = model.loss(x, t, p, seed=step)
            grads = torch.autograd.grad(loss, model.matrices() + model.others())
            opt.step_math(grads[:len(whiten)])
            rest.step_math(grads[len(whiten):])
            losses.append(loss.detach().item())
        if step % 10 == 0:
            log(f"step {step:4d}  loss {losses[-1]:.4f}")
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    for name, value in (("steps", 60), ("dim", 256), ("layers", 2), ("vocab", 4096), ("batch", 16), ("tokens", 128)):
        ap.add_argument("--" + name, type=int, default=value)
    ap.add_argument("--p", type=float, default=0.1)
    ap.add_argument("--window", type=int, default=None)
    ap.add_argument("--sinks", type=int, default=0)
    a = ap.parse_args()
    out = train(**vars(a))
    print(json.dumps({"loss_first_last": [round(out[0], 4), round(sum(out[-5:]) / min(5, len(out)), 4)], **vars(a)}))
