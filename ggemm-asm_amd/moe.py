"""What an MoE layer does around its grouped products, as torch ops over the C ABI (include/ggemm_moe.h).

* ``route_experts``   -- the experts of each token and their weights from the router's logits
* ``plan_dispatch``   -- the choices ordered by expert: the group offsets that the grouped products take and the
  row of every choice
* ``dispatch_tokens`` -- the tokens' rows copied into that order
* ``combine_tokens``  -- each token's weighted sum over its experts' rows, added to a residual

The reference's harness makes its group offsets on the host and has none of these (reference bench.py:196-209).
``route_experts``, ``dispatch_tokens`` and ``combine_tokens`` are differentiable. Every launch goes through
libggemm_vark.so on torch's current stream; nothing synchronises, so all of it can be captured in a HIP graph;
there is no CPU path.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from ._tensors import on_gpu as _on_gpu, once_differentiable, row_stride as _stride, tracked

_IN = {torch.bfloat16: 0, torch.float32: 1}
_SCORES = {"softmax": 0, "sigmoid": 1}
MAX_EXPERTS = 1024      # of a router
MAX_TOP_K = 64
MAX_GROUPS = 2047       # of a plan
_PLAN_ALONE = 2048      # GGEMM_MOE_PLAN_ALONE: plans up to so many choices need no workspace


class DispatchPlan(NamedTuple):
    """Where the choices of T tokens went: ``group_offs`` int64 [G + 1], the rows of each expert, and ``slots`` int32
    [T, k], the row of each choice or -1. Rows of one expert are in the order of their tokens."""
    group_offs: torch.Tensor
    slots: torch.Tensor


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A 2-D tensor whose rows are contiguous and do not overlap (a copy where they are not)."""
    if t.stride(1) != 1 and t.shape[1] > 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        return t.contiguous()
    return t


# --------------------------------------------------------------------------- routing

def _route(logits, top_k, score, bias, num_groups, top_groups, group_best, renormalize, scale):
    T, E = logits.shape
    dev = logits.device
    weights = torch.empty((T, top_k), dtype=torch.float32, device=dev)
    experts = torch.empty((T, top_k), dtype=torch.int32, device=dev)
    if T:
        _lib.launch("ggemm_moe_route", dev, E | top_k | num_groups | top_groups, logits.data_ptr(), _IN[logits.dtype], T,
                    E, _stride(logits), top_k, score, None if bias is None else bias.data_ptr(), num_groups, top_groups,
                    group_best, renormalize, scale, weights.data_ptr(), experts.data_ptr())
    return weights, experts


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, *args):
        top_k, score, bias, num_groups, top_groups, group_best, renormalize, scale = args
        weights, experts = _route(logits, *args)
        ctx.save_for_backward(logits, experts)
        ctx.args = score, renormalize, scale
        ctx.mark_non_differentiable(experts)
        ctx.set_materialize_grads(False)              # no zeros made for the experts, which have no gradient
        return weights, experts

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, _):
        if dweights is None:
            return (None,) * 9
        logits, experts = ctx.saved_tensors
        score, renormalize, scale = ctx.args
        T, E = logits.shape
        dlogits = torch.empty((T, E), dtype=logits.dtype, device=logits.device)
        if T:
            dweights = dweights.contiguous()
            k = experts.shape[1]
            _lib.launch("ggemm_moe_route_backward", logits.device, E | k, dweights.data_ptr(), logits.data_ptr(),
                        _IN[logits.dtype], T, E, _stride(logits), k, score, renormalize, scale, experts.data_ptr(),
                        dlogits.data_ptr())
        return (dlogits,) + (None,) * 8


def route_experts(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: torch.Tensor | None = None,
                  num_groups: int = 1, top_groups: int | None = None, group_best: int = 2, renormalize: bool = True,
                  scale: float = 1.0):
    """``(weights, experts)`` of each token: fp32 and int32 [T, top_k], from router logits bf16 / fp32 [T, E].

    ``score``: "softmax" over the E logits or "sigmoid" of each. Experts are taken by their key, the largest first and
    equal keys by the lower index: score + ``bias`` (fp32 [E], moved by a balancing rule, not by gradients) with a
    bias, the score with groups, else the logit. ``num_groups`` > 1: of the groups of E / num_groups consecutive
    experts only the ``top_groups`` whose ``group_best`` (1 or 2) largest keys have the largest sum are looked at.
    Weights are ``scale`` times the score, divided by the sum over the token's experts if ``renormalize`` (a softmax
    over the taken logits for softmax). Experts whose logit or key is -inf are never taken: a token with fewer than
    top_k others has -1 with weight 0 in the last places. NaN counts as larger than any number. Gradients of the
    weights flow to the logits."""
    if logits.dim() != 2 or logits.dtype not in _IN:
        raise TypeError("logits must be a bf16 or fp32 [T, E] tensor")
    _on_gpu(logits, "routing")
    E = logits.shape[1]
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"routing takes 1 to {MAX_EXPERTS} experts, got {E}")
    if not 1 <= top_k <= min(E, MAX_TOP_K):
        raise ValueError(f"top_k must be in [1, {min(E, MAX_TOP_K)}], got {top_k}")
    if score not in _SCORES:
        raise ValueError(f"score must be 'softmax' or 'sigmoid', got {score!r}")
    top_groups = num_groups if top_groups is None else top_groups
    if num_groups < 1 or E % num_groups or not 1 <= top_groups <= num_groups:
        raise ValueError(f"{E} experts in {num_groups} groups, {top_groups} of them taken: not possible")
    if group_best not in (1, 2) or num_groups > 1 and E // num_groups < group_best:
        raise ValueError("group_best must be 1 or 2 and no more than the experts of a group")
    if bias is not None:
        if bias.dtype != torch.float32 or tuple(bias.shape) != (E,) or bias.device != logits.device:
            raise ValueError(f"bias must be fp32 [{E}] on the logits' device")
        bias = bias.detach().contiguous()
    args = (top_k, _SCORES[score], bias, num_groups, top_groups, group_best, int(bool(renormalize)), float(scale))
    if tracked(logits):
        return _Route.apply(_rows(logits), *args)
    return _route(_rows(logits), *args)


# --------------------------------------------------------------------------- order, copy and sum of rows

def plan_dispatch(experts: torch.Tensor, num_experts: int) -> DispatchPlan:
    """The order of the choices ``experts`` (int32 [T, k]) by expert: a ``DispatchPlan`` for G = num_experts groups.
    Choices outside [0, num_experts), as ``route_experts``' -1, get no row (slot -1). A rank that holds some of the
    experts passes ``experts - first``. The rows of a plan are [T * k, H], those from group_offs[G] on unused."""
    if experts.dtype != torch.int32 or experts.dim() != 2:
        raise TypeError("experts must be an int32 [T, k] tensor")
    if not 1 <= num_experts <= MAX_GROUPS:
        raise ValueError(f"num_experts must be in [1, {MAX_GROUPS}], got {num_experts}")
    _on_gpu(experts, "the dispatch plan")
    experts = experts.contiguous()
    dev, n = experts.device, experts.numel()
    offs = torch.empty(num_experts + 1, dtype=torch.int64, device=dev)
    slots = torch.empty_like(experts)
    ws = None
    if n > _PLAN_ALONE:
        ws = torch.empty(_lib.load().ggemm_moe_plan_workspace(n, num_experts), dtype=torch.int32, device=dev)
    _lib.launch("ggemm_moe_plan", dev, num_experts, experts.data_ptr(), n, num_experts, offs.data_ptr(),
                slots.data_ptr(), None if ws is None else ws.data_ptr())
    return DispatchPlan(offs, slots)


def _check_plan(plan: DispatchPlan, dev):
    offs, slots = plan
    if offs.dtype != torch.int64 or offs.dim() != 1 or not 2 <= offs.numel() <= MAX_GROUPS + 1:
        raise ValueError("the plan's group_offs must be int64 [G + 1]")
    if slots.dtype != torch.int32 or slots.dim() != 2:
        raise ValueError("the plan's slots must be int32 [T, k]")
    if offs.device != dev or slots.device != dev:
        raise ValueError("all tensors must be on the same device")
    return offs.contiguous(), slots.contiguous()


def _dispatch(x, offs, slots, row_align):
    T, H = x.shape
    k, item = slots.shape[1], x.element_size()
    if row_align and H * item % row_align:
        pitch = -(-H * item // row_align) * row_align
        rows = torch.empty((T * k, pitch // item), dtype=x.dtype, device=x.device)[:, :H]
    else:
        rows = torch.empty((T * k, H), dtype=x.dtype, device=x.device)
    if rows.numel():
        G = offs.numel() - 1
        _lib.launch("ggemm_moe_dispatch", x.device, G | k, x.data_ptr(), H * item, _stride(x) * item, T, k,
                    slots.data_ptr(), offs.data_ptr(), G, rows.data_ptr(), rows.stride(0) * item, T * k)
    return rows


def _combine(y, slots, weights, residual):
    (M, H), (T, k) = y.shape, slots.shape
    out = torch.empty((T, H), dtype=y.dtype, device=y.device)
    if out.numel():
        # a y without rows has a null pointer: every choice is without a row then, and none is read
        yp = y.data_ptr() if M else out.data_ptr()
        _lib.launch("ggemm_moe_combine", y.device, H | k, yp, _IN[y.dtype], _stride(y), M, slots.data_ptr(), T, k,
                    None if weights is None else weights.data_ptr(), None if residual is None else residual.data_ptr(),
                    0 if residual is None else _stride(residual), H, out.data_ptr(), H)
    return out


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, offs, slots, row_align):
        ctx.save_for_backward(slots)
        return _dispatch(x, offs, slots, row_align)

    @staticmethod
    @once_differentiable
    def backward(ctx, drows):
        slots, = ctx.saved_tensors
        return _combine(_rows(drows), slots, None, None), None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, residual, offs, slots):
        need_y, need_w, _ = ctx.needs_input_grad[:3]      # y is read for the weights' gradient alone, the weights for y's
        ctx.save_for_backward(y if need_w else None, weights if need_y else None, offs, slots)
        ctx.y_shape = y.shape
        return _combine(y, slots, weights, residual)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        y, weights, offs, slots = ctx.saved_tensors
        need_y, need_w, need_r = ctx.needs_input_grad[:3]
        (M, H), (T, k), dev = ctx.y_shape, slots.shape, slots.device
        dres = dout if need_r else None
        dout = _rows(dout)
        dy = torch.empty((M, H), dtype=dout.dtype, device=dev) if need_y else None
        dw = torch.empty((T, k), dtype=torch.float32, device=dev) if need_w else None
        if T and H and M:
            G = offs.numel() - 1
            _lib.launch("ggemm_moe_combine_backward", dev, H | k | G, dout.data_ptr(), _IN[dout.dtype], _stride(dout),
                        None if y is None else y.data_ptr(), H if y is None else _stride(y), M, slots.data_ptr(), T, k,
                        None if weights is None else weights.data_ptr(), offs.data_ptr(), G, H,
                        None if dy is None else dy.data_ptr(), H, None if dw is None else dw.data_ptr())
        else:
            dy, dw = (None if t is None else t.zero_() for t in (dy, dw))
        return dy, dw, dres, None, None


def dispatch_tokens(x: torch.Tensor, plan: DispatchPlan, row_align: int | None = None) -> torch.Tensor:
    """``rows[plan.slots[t, j]] = x[t]``: [T * k, H] of x's type, rows from ``plan.group_offs[G]`` on zero.

    x: [T, H] bf16 / fp32 (differentiable: the sum over the token's rows), or fp8 / bytes: a batch quantized once and
    copied afterwards moves half the bytes of one copied first. ``row_align=128`` starts the rows on 128-byte lines
    (a view of a padded buffer, the padding not written), as the grouped products read them best."""
    if x.dim() != 2:
        raise ValueError("x must be a [T, H] tensor")
    _on_gpu(x, "the dispatch")
    offs, slots = _check_plan(plan, x.device)
    if slots.shape[0] != x.shape[0]:
        raise ValueError(f"x holds {x.shape[0]} tokens, the plan {slots.shape[0]}")
    if row_align is not None and (row_align < 1 or row_align % x.element_size()):
        raise ValueError("row_align must be a multiple of the element size")
    if tracked(x):
        if x.dtype not in _IN:
            raise TypeError(f"gradients flow to bf16 or fp32 tokens only, got {x.dtype}")
        return _Dispatch.apply(_rows(x), offs, slots, row_align)
    return _dispatch(_rows(x), offs, slots, row_align)


def combine_tokens(y: torch.Tensor, plan: DispatchPlan, weights: torch.Tensor | None = None,
                   residual: torch.Tensor | None = None) -> torch.Tensor:
    """``out[t] = residual[t] + sum_j weights[t, j] * y[plan.slots[t, j]]``: [T, H] of y's type, summed in fp32 in the
    order of j and rounded once. y: bf16 / fp32 [M, H]; weights: fp32 [T, k] (ones without); residual: [T, H] of y's
    type. Choices without a row have no term. Differentiable by y (rows from ``plan.group_offs[G]`` on get zero),
    weights and residual."""
    if y.dim() != 2 or y.dtype not in _IN:
        raise TypeError("y must be a bf16 or fp32 [M, H] tensor")
    _on_gpu(y, "the combination")
    offs, slots = _check_plan(plan, y.device)
    T, k = slots.shape
    if weights is not None:
        if weights.dtype != torch.float32 or tuple(weights.shape) != (T, k) or weights.device != y.device:
            raise ValueError(f"weights must be fp32 [{T}, {k}] on y's device")
        weights = weights.contiguous()
    if residual is not None:
        if residual.dtype != y.dtype or tuple(residual.shape) != (T, y.shape[1]) or residual.device != y.device:
            raise ValueError(f"residual must be {y.dtype} [{T}, {y.shape[1]}] on y's device")
        residual = _rows(residual)
    if tracked(y, weights, residual):
        return _Combine.apply(_rows(y), weights, residual, offs, slots)
    return _combine(_rows(y), slots, weights, residual)
