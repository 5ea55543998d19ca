"""Layer norm and the gated feed-forward block on torch CUDA tensors, with their
backward passes.

Each call checks shapes, types and strides, allocates the outputs, enqueues the
kernels on the current stream of the inputs' device and raises on a non-zero
status (_torch_ops.so, which calls the C ABI). Matrices have a unit column
stride and any row stride.

No call records anything for torch's autograd, whatever its inputs require:
gradients come from the *_backward functions.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._capi import torch_ops as _torch_ops
from .vocab import _DT


class LayerNorm(NamedTuple):
    y: torch.Tensor
    mean: torch.Tensor  # float32 [rows]
    rstd: torch.Tensor  # float32 [rows]


def layer_norm(x, weight=None, bias=None, eps=1e-5, out_dtype=None, out=None) -> LayerNorm:
    """Layer norm of the rows of x: (x - mean) * rstd * weight + bias. The result
    has x's type, or out_dtype (16 bits for float32 x). weight and bias: both of
    one type, or None. out: where to write it (may be x itself, but not overlap
    it otherwise)."""
    if out_dtype is not None and out_dtype not in _DT:
        raise ValueError("out_dtype: expected float32, bfloat16 or float16")
    return LayerNorm(*_torch_ops.layer_norm(x, weight, bias, eps, -1 if out_dtype is None else _DT[out_dtype], out))


def layer_norm_backward(dy, x, mean, rstd, weight=None, need_weight=True, need_bias=False, out=None):
    """Gradients of layer_norm with respect to x, weight and bias (the latter two
    in weight's type, float32 without one; None where not needed), from its mean
    and rstd. out: where to write dx (may be dy or x itself, but not overlap them
    otherwise)."""
    return _torch_ops.layer_norm_backward(dy, x, mean, rstd, weight, bool(need_weight), bool(need_bias), out)


ACTIVATIONS = {"gelu": 0, "gelu_tanh": 1, "silu": 2}


def _activation(name):
    act = ACTIVATIONS.get(name)
    if act is None:
        raise ValueError(f"activation: expected one of {', '.join(ACTIVATIONS)}")
    return act


def gated_ff(x, w_in, w_out, activation="gelu", save=False):
    """The gated feed-forward block (act(a) * b) @ w_out.T with [a | b] = x @
    w_in.T: x [rows, hidden], w_in [2 * inner, hidden] (the activated rows
    first), w_out [out, inner], all bfloat16 or all float16. activation: "gelu",
    "gelu_tanh" or "silu". save=True: (y, what gated_ff_backward needs).

    act(a) * b is rounded to the operands' type before the second product. One
    row, or up to four where the weights are few, keeps it in float32 unless save
    is asked for, so that its y may differ in the last place from the same row's
    in a larger call."""
    r = _torch_ops.gated_ff(x, w_in, w_out, _activation(activation), bool(save))
    return r if save else r[0]


def gated_ff_backward(dy, x, w_in, w_out, saved, activation="gelu", need_input=True, need_in=True, need_out=True):
    """Gradients of gated_ff with respect to x, w_in and w_out, in their type
    (None where not needed), from dy and what the forward with the same operands
    saved. The gradient of [a | b] in between is rounded to the operands' type."""
    return _torch_ops.gated_ff_backward(dy, x, w_in, w_out, saved, _activation(activation), bool(need_input), bool(need_in),
                                        bool(need_out))
