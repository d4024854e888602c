"""The gated first half of a feed-forward block, with its backward pass.

The kernels and their checks of arguments are in the compiled extension; this is what joins them to
PyTorch's autograd.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

__all__ = ["gated_linear"]


def _ext():
    from . import _cmpext3

    return _cmpext3


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, activation):
        out, gate, up = _ext()._gated_forward(x, w_gate, w_up, activation, True)
        ctx.activation = activation
        ctx.save_for_backward(x, w_gate, w_up, gate, up)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return (*_ext()._gated_backward(grad, *ctx.saved_tensors, ctx.activation, *ctx.needs_input_grad[:3]), None)


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """act(x @ w_gate.T) * (x @ w_up.T) in one kernel: x [..., K], weights [N, K], all float16 or all
    bfloat16; sums and the activation in fp32, rounded once.

    activation: "silu", "gelu" (by the error function), "gelu_tanh" or "relu".

    Differentiable once in all three tensors.  For the backward pass x, the weights and both products
    (in float32, 8 bytes for each result) are kept; where no input needs a gradient nothing is.  Weights may be
    the two halves of one tensor; rows of whole 16 bytes are read in place, others are copied first.
    Under graph capture the inputs' leaves must not be held by a graph of another stream (refused).
    """
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad):
        _ext()._check_capture([x, w_gate, w_up])
        return _GatedLinear.apply(x, w_gate, w_up, activation)
    return _ext()._gated_forward(x, w_gate, w_up, activation, False)[0]
