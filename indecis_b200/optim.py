"""AdamW over many tensors at once on torch CUDA tensors, moments in 32 or in 8
bits (ig_adamw_step), as a function and as an object that keeps the moments.

Nothing is copied to the device and nothing waits for it: the step count, a
gradient scale and a flag that skips the step are read from the device when the
step runs, so a captured step takes the next one at every replay.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._capi import torch_ops as _torch_ops

BLOCK = 256  # elements of a tensor that share a scale in 8 bits


class Moment8(NamedTuple):
    """A tensor's moment in 8 bits: codes times the scale of their 256 elements."""
    codes: torch.Tensor   # float8_e4m3fn, the parameter's shape
    scales: torch.Tensor  # float32 [ceil(n / 256)]

    def values(self):
        """The moment (exp_avg), or the root of it (exp_avg_sq), in float32."""
        n = self.codes.numel()
        return (self.codes.float().reshape(-1) * self.scales.repeat_interleave(BLOCK)[:n]).view(self.codes.shape)


torch.serialization.add_safe_globals([Moment8])  # torch.load takes a saved state_dict as it comes


def new_moment(param, bits=32):
    """A moment of zeros for param, in 32 or 8 bits."""
    if bits == 32:
        return torch.zeros(param.shape, dtype=torch.float32, device=param.device)
    if bits != 8:
        raise ValueError("moments are held in 32 or in 8 bits")
    return Moment8(torch.zeros(param.shape, dtype=torch.float8_e4m3fn, device=param.device),
                   torch.zeros(-(-param.numel() // BLOCK), dtype=torch.float32, device=param.device))


def adamw_step(params, grads, exp_avg, exp_avg_sq, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
               copies=None, grad_scale=None, skip=None):
    """One AdamW step in place over lists of contiguous tensors.

    params, grads: float32, bfloat16 or float16, types free. exp_avg, exp_avg_sq:
    float32 tensors, or (codes, scales) pairs (Moment8) for all of them. step:
    int32, one value, the steps taken so far; the call adds 1. weight_decay: one
    number or one for each tensor. copies: 16-bit tensors that receive the new
    parameters, or None. grad_scale, skip: float32, one value each: the factor of
    every gradient, and where not 0 nothing changes (an overflow found elsewhere).
    No two tensors that are written may share memory. A gradient that is None
    leaves its tensor out (its moments may be None too)."""
    _torch_ops.adamw_step(params, grads, exp_avg, exp_avg_sq, step, lr, betas[0], betas[1], eps, weight_decay, copies, grad_scale,
                          skip)


class AdamW:
    """Keeps the moments and the step count of a list of parameters.

    opt = AdamW(params, lr=3e-4, bits=8); opt.step(grads). lr may be set between
    steps (opt.lr). copies: 16-bit tensors that follow the parameters."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, bits=32, copies=None):
        self.params = list(params)
        if not self.params:
            raise ValueError("params: expected one tensor at least")
        self.copies = list(copies) if copies is not None else None
        self.lr, self.betas, self.eps, self.weight_decay, self.bits = lr, betas, eps, weight_decay, bits
        self.exp_avg = [new_moment(p, bits) for p in self.params]
        self.exp_avg_sq = [new_moment(p, bits) for p in self.params]
        self.steps = torch.zeros(1, dtype=torch.int32, device=self.params[0].device)

    def step(self, grads=None, grad_scale=None, skip=None):
        """One step with the given gradients (default: the parameters' .grad)."""
        adamw_step(self.params, [p.grad for p in self.params] if grads is None else grads, self.exp_avg, self.exp_avg_sq,
                   self.steps, self.lr, self.betas, self.eps, self.weight_decay, self.copies, grad_scale, skip)

    def state_dict(self):
        """The moments and the count (the tensors themselves: clone what is kept)."""
        return {"exp_avg": self.exp_avg, "exp_avg_sq": self.exp_avg_sq, "steps": self.steps}

    def load_state_dict(self, state):
        """Copies the values of a state_dict of the same parameters."""
        def pieces(m):
            return [m] if isinstance(m, torch.Tensor) else list(m)
        mine, theirs = ([t for k in ("exp_avg", "exp_avg_sq") for m in s[k] for t in pieces(m)] + [s["steps"]]
                        for s in (self.state_dict(), state))
        if [(t.shape, t.dtype) for t in mine] != [(t.shape, t.dtype) for t in theirs]:
            raise ValueError("state: expected moments of the same sizes and types")
        for a, b in zip(mine, theirs):
            a.copy_(b)
