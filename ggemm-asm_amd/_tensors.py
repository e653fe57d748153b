"""What the ops ask of the tensors they are given, and of autograd."""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch
import torch.autograd.forward_ad as fwAD
from torch.autograd.function import once_differentiable as _once_differentiable


class MXTensor(NamedTuple):
    """Rows in blocks of 32 that share a power of two: ``q`` float8_e4m3fn [.., K], or uint8 [.., K / 2] with two e2m1
    values in a byte, the even column in its low half; ``scales`` uint8 [.., ceil(K / 32)], a block's power of two as its
    exponent + 127 (255: NaN)."""
    q: torch.Tensor
    scales: torch.Tensor


MX_BLOCK = 32                    # values that share a scale


def mx_columns(t: MXTensor, what: str) -> tuple[int, int]:
    """(format code, columns) of a microscaled tensor whose parts fit each other."""
    q, scales = t
    if q.dtype == torch.float8_e4m3fn:
        code, cols = 0, q.shape[-1]
    elif q.dtype == torch.uint8:
        code, cols = 1, 2 * q.shape[-1]
    else:
        raise TypeError(f"{what} must hold float8_e4m3fn values or uint8 pairs of e2m1, got {q.dtype}")
    if scales.dtype != torch.uint8 or scales.shape != q.shape[:-1] + (-(-cols // MX_BLOCK),):
        raise ValueError(f"{what}'s scales must be uint8 {list(q.shape[:-1]) + [-(-cols // MX_BLOCK)]}")
    if scales.device != q.device:
        raise ValueError(f"{what}'s values and scales must be on the same device")
    return code, cols


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
