"""AdamW on the HIP kernels (include/psgdk.h, level 3): the step of what a Kron preconditioner does not suit (embeddings, norm
weights, biases, gates), or of a whole model.

    AdamW        the optimizer, in KronWhiten's manner
    adamw_step   one step over tensors and states that the caller holds
    adamw_state  zeroed states in 32 or 8 bits

CUDA (HIP) tensors in float32 or bfloat16, on torch's current stream, all tensors in one launch for each 128. No counterparts in
the reference.
"""
import ctypes as C
import math

import torch

from . import _lib as L
from .train import _run_ws

__all__ = ["AdamW", "adamw_state", "adamw_step"]

_BLOCK = 256  # elements that share a scale
_CODES, _SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _tables(params, grads, ms, vs):
    """The host arrays of psgdk_adamw_t for lists of tensors, checked (csrc/tables.cpp): (their buffer, the states' bits, copies of
    gradients that had to be made contiguous)."""
    buf = (C.c_int64 * (8 * len(params)))()
    return (buf, *L.tables().adamw(params, grads, ms, vs, C.addressof(buf), len(buf)))


def _check_numbers(step, lr, betas, eps, weight_decay, max_norm):
    if not 1 <= step <= 1 << 32:
        raise ValueError(f"step = {step}: counts from 1")
    if not (math.isfinite(lr) and math.isfinite(weight_decay)):
        raise ValueError(f"lr = {lr}, weight_decay = {weight_decay}: must be finite")
    if not all(0 <= b < 1 for b in betas) or len(betas) != 2:
        raise ValueError(f"betas = {betas}: two numbers in 0..1, below 1")
    if not eps >= 0:
        raise ValueError(f"eps = {eps}: must be >= 0")
    if max_norm is not None and not max_norm > 0:
        raise ValueError(f"max_norm = {max_norm}: must be positive, or None")


def _launch(params, grads, ms, vs, step, lr, betas, eps, weight_decay, max_norm, seed):
    buf, bits, keep = _tables(params, grads, ms, vs)
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("psgd_pro_amd: an AdamW step is not captured into a graph (its number would stay the same)")
    norm = torch.empty((), device=params[0].device, dtype=torch.float32) if max_norm is not None else None
    at, n = C.addressof(buf), 8 * len(params)
    scales = (at + 6 * n, at + 7 * n) if bits == 8 else (None, None)
    a = L.AdamW(len(params), bits, at, at + n, at + 2 * n, at + 3 * n, at + 4 * n, at + 5 * n, *scales, lr, betas[0], betas[1], eps,
                weight_decay, max_norm or 0.0, step, seed, None if norm is None else norm.data_ptr())
    _run_ws(params[0], L.lib().psgdk_adamw, C.byref(a))
    L.tables().changed(params)  # (as by torch's own in-place operations)
    return norm


def adamw_state(like, bits=32):
    """A zeroed first or second moment for the parameter `like`: float32 of its shape, or (codes, scales) with 8 bits: e4m3 codes,
    one for each element, and a power-of-two scale for each 256 of them. A first moment is codes * scales, a second moment its
    square."""
    if bits == 32:
        return torch.zeros(like.shape, device=like.device, dtype=torch.float32)
    if bits != 8:
        raise ValueError(f"bits = {bits}: 8 or 32")
    n = like.numel()
    return (torch.zeros(n, device=like.device, dtype=torch.uint8).view(_CODES),
            torch.zeros(-(-n // _BLOCK), device=like.device, dtype=torch.uint8).view(_SCALES))


@torch.no_grad()
def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
               max_norm=None, seed=0):
    """One AdamW step, in place, over lists of parameters, their gradients (same shapes and dtypes) and their states:

        g = gradient * min(1, max_norm / norm of all gradients)   (max_norm None: the gradient)
        m = beta1 m + (1 - beta1) g;   v = beta2 v + (1 - beta2) g^2
        p = (1 - lr weight_decay) p - lr m / (1 - beta1^step) / (sqrt(v / (1 - beta2^step)) + eps)

    States are adamw_state's, all of one kind: float32 tensors, or with 8 bits (codes, scales) of the first moment and of the
    second's root. Codes are rounded up or down by chance, by Philox4x32-10 under (seed, step, the tensor's place in the list), so
    that an average does not stop where a step's change is less than half a code; the update takes the values before rounding.
    Gradients from 2^64 on: with 32 bits v is infinite and the element only decays from then on; with 8 bits, which hold the root,
    they count as any other up to 2^125. An infinity or NaN makes NaN of its 256 elements' states with 8 bits.
    bfloat16 parameters are rounded to nearest. Tensors may begin anywhere in their storage, parameters and states are contiguous.
    Returns the gradients' norm before clipping (a 0-d float32 tensor) where max_norm is given. Capture into a graph is refused."""
    _check_numbers(step, lr, betas, eps, weight_decay, max_norm)
    return _launch(list(params), list(grads), list(exp_avgs), list(exp_avg_sqs), int(step), float(lr), tuple(map(float, betas)),
                   float(eps), float(weight_decay), max_norm, int(seed) & (2 ** 64 - 1))


class AdamW:
    """AdamW over the parameters that require gradients, in KronWhiten's manner: mutable attributes lr_params, betas, eps,
    weight_decay and max_norm, step(closure) returning the closure's value, step_math(grads), state_dict() and load_state_dict().

    max_norm: clip by the norm of all of them (norm: the last step's, before clipping, on the device). state_bits: 32, or 8 (e4m3
    codes with a power-of-two scale for each 256 elements, see adamw_step). seed: of the 8-bit states' rounding; None draws one
    from torch's CPU generator. Beside KronWhiten, take the gradients of all parameters and give each optimizer its own:

        grads = torch.autograd.grad(loss, matrices + others)
        kron.step_math(grads[:len(matrices)]); adamw.step_math(grads[len(matrices):])"""

    def __init__(self, params_with_grad, lr_params=0.001, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, max_norm=None, *,
                 state_bits=32, seed=None):
        params = [params_with_grad] if isinstance(params_with_grad, torch.Tensor) else params_with_grad
        self._params_with_grad = [p for p in params if p.requires_grad]
        if not self._params_with_grad:
            raise ValueError("no parameters that require gradients")
        _check_numbers(1, lr_params, betas, eps, weight_decay, max_norm)
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits = {state_bits}: 8 or 32")
        self.lr_params, self.betas, self.eps, self.weight_decay, self.max_norm = lr_params, tuple(betas), eps, weight_decay, max_norm
        self.norm = None
        self._bits = state_bits
        self._seed = (int(torch.randint(2 ** 62, ())) if seed is None else int(seed)) & (2 ** 64 - 1)
        self._step = 0
        self._ms = [adamw_state(p, state_bits) for p in self._params_with_grad]
        self._vs = [adamw_state(p, state_bits) for p in self._params_with_grad]
        _tables(*([p.detach() for p in self._params_with_grad],) * 2, self._ms, self._vs)  # (refuses what a step would)

    @torch.no_grad()
    def step_math(self, grads):
        """One step with the gradients given."""
        _check_numbers(self._step + 1, self.lr_params, self.betas, self.eps, self.weight_decay, self.max_norm)
        norm = _launch(self._params_with_grad, list(grads), self._ms, self._vs, self._step + 1, float(self.lr_params),
                       tuple(map(float, self.betas)), float(self.eps), float(self.weight_decay), self.max_norm, self._seed)
        self._step += 1
        if norm is not None:
            self.norm = norm

    @torch.no_grad()
    def step(self, closure):
        """Evaluates the closure, takes the gradients with torch.autograd.grad, steps, and returns what the closure returned."""
        with torch.enable_grad():
            closure_returns = closure()
            loss = closure_returns if isinstance(closure_returns, torch.Tensor) else closure_returns[0]
            grads = torch.autograd.grad(loss, self._params_with_grad)
        self.step_math(grads)
        return closure_returns

    def moments(self, i):
        """(m, v) of parameter i in float32, in its shape (copies)."""
        shape = self._params_with_grad[i].shape
        if self._bits == 32:
            return self._ms[i].clone(), self._vs[i].clone()
        m, r = (c.float() * s.float().repeat_interleave(_BLOCK)[:c.numel()] for c, s in (self._ms[i], self._vs[i]))
        return m.view(shape), r.square_().view(shape)

    def state_dict(self):
        copy = lambda s: s.clone() if self._bits == 32 else tuple(t.clone() for t in s)  # noqa: E731
        return dict(version=1, state_bits=self._bits, step=self._step, seed=self._seed,
                    hyper=dict(lr_params=self.lr_params, betas=self.betas, eps=self.eps, weight_decay=self.weight_decay,
                               max_norm=self.max_norm),
                    exp_avgs=[copy(s) for s in self._ms], exp_avg_sqs=[copy(s) for s in self._vs])

    def load_state_dict(self, st):
        if st["state_bits"] != self._bits:
            raise ValueError(f"the state has {st['state_bits']} bits, this optimizer's {self._bits}")
        pairs = []
        for mine, saved in ((self._ms, st["exp_avgs"]), (self._vs, st["exp_avg_sqs"])):
            if len(mine) != len(saved):
                raise ValueError(f"the state is of {len(saved)} parameters, this optimizer has {len(mine)}")
            for i, (a, b) in enumerate(zip(mine, saved)):
                for x, y in ((a, b),) if self._bits == 32 else zip(a, b):
                    if x.shape != y.shape or x.dtype != y.dtype:
                        raise ValueError(f"state for parameter {i} does not match its shape")
                    pairs.append((x, y))
        for k, v in st["hyper"].items():
            setattr(self, k, v)
        self._step, self._seed = st["step"], st["seed"]
        for x, y in pairs:
            (x if x.dtype == torch.float32 else x.view(torch.uint8)).copy_(y if y.dtype == torch.float32 else y.view(torch.uint8))
