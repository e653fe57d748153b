"""What the ops ask of the tensors they are given, and of autograd."""
from __future__ import annotations

import functools

import torch
import torch.autograd.forward_ad as fwAD
from torch.autograd.function import once_differentiable as _once_differentiable


def on_gpu(t: torch.Tensor, what: str) -> None:
    if t.device.type != "cuda":
        raise ValueError(f"{what} runs on a gfx950 GPU only (tensors are on {t.device})")


def row_stride(t: torch.Tensor) -> int:
    """Row stride of a 2-D tensor; where there is one row its own is arbitrary and not used."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def once_differentiable(backward):
    """torch's once_differentiable, entered only under create_graph=True: everywhere else a backward pass runs without
    grad mode anyway, where torch's wrapper would cost 4 us (of the 86 of a routing step and its gradient)."""
    refusing = _once_differentiable(backward)

    @functools.wraps(backward)
    def wrapper(ctx, *args):
        return refusing(ctx, *args) if torch.is_grad_enabled() else backward(ctx, *args)

    return wrapper


def tracked(*tensors: torch.Tensor | None) -> bool:
    """Whether autograd has to see a call on these tensors (None for none): one requires a gradient, or has a
    forward-mode tangent, which the ops have no rule for and their autograd functions refuse."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    # the level is asked first: outside of dual levels, nearly always, no tensor has to be
    return fwAD._current_level >= 0 and any(t is not None and fwAD.unpack_dual(t).tangent is not None for t in tensors)
