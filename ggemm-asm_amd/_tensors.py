"""What the ops ask of the tensors they are given, and of autograd."""
from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable as _once_differentiable


def once_differentiable(backward):
    """torch's once_differentiable, entered only under create_graph=True: everywhere else a backward pass runs without
    grad mode anyway, where torch's wrapper would cost 4 us (of the 86 of a routing step and its gradient)."""
    refusing = _once_differentiable(backward)

    @functools.wraps(backward)
    def wrapper(ctx, *args):
        return refusing(ctx, *args) if torch.is_grad_enabled() else backward(ctx, *args)

    return wrapper
