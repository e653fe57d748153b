"""A whole MoE layer: routing, dispatch, the experts' two FP8 products and the combination.

``moe_layer_fp8`` is how the package's operators are meant to follow one another; a model with another order of steps
calls them one by one. The reference's harness runs the products alone, on random rows (reference bench.py:196-268).
"""
from __future__ import annotations

import torch

from ._tensors import tracked
from .autograd import FP8DelayedScaling, FP8WeightCache, grouped_linear_fp8
from .moe import combine_tokens, dispatch_tokens, plan_dispatch, route_experts
from .product import _rows16, grouped_gemm_fp8_bias_act
from .quant import quantize_fp8_tensorwise

_LINE = 128


def _weight(w, cache):
    if cache is not None:
        qw, _, sw = cache.get(w, False)
        return qw, sw
    qw, sw, _ = quantize_fp8_tensorwise(w.contiguous(), "e4m3", row_align=_LINE)
    return qw, sw


def moe_layer_fp8(x: torch.Tensor, logits: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, top_k: int, *,
                  bias_up: torch.Tensor | None = None, bias_down: torch.Tensor | None = None,
                  activation: str | None = "swiglu", slope: float = 1.0, limit: float | None = None,
                  shift: float = 0.0, residual: torch.Tensor | None = None, routing: dict | None = None,
                  main_grads: tuple | None = None, weight_caches: tuple[FP8WeightCache, FP8WeightCache] | None = None,
                  scalings: tuple[FP8DelayedScaling, FP8DelayedScaling] | None = None) -> torch.Tensor:
    """``residual + sum_j weight_j * expert_j(x)`` of every token, [T, H] bf16.

    x: bf16 [T, H]; logits: the router's, [T, E]; w_up: [E, N, H] and w_down: [E, H, I], bf16 / fp32, I = N / 2 for
    "swiglu" and N otherwise; biases [E, N] and [E, H]. ``routing``: options of ``route_experts``; ``slope``, ``limit``,
    ``shift``: of the activation; ``main_grads``, ``weight_caches``, ``scalings``: those of ``grouped_linear_fp8``, for
    the two products.

    With gradients: rows are dispatched in bf16 and the products are the autograd layer's. Without: x is quantized once
    and its fp8 rows dispatched, half the bytes of bf16 ones, and nothing is kept for a backward pass (delayed scaling
    is a training recipe and is not used there). Either way x's scale is that of the tokens that go to an expert:
    what a masked token (all logits -inf) holds reaches no other token."""
    if x.dim() != 2 or x.dtype != torch.bfloat16:
        raise TypeError("x must be a bf16 [T, H] tensor")
    if logits.dim() != 2 or logits.shape[0] != x.shape[0] or logits.shape[1] != w_up.shape[0]:
        raise ValueError(f"logits must be [{x.shape[0]}, {w_up.shape[0]}]")
    if w_down.shape[0] != w_up.shape[0] or w_down.shape[1] != x.shape[1]:
        raise ValueError("w_up and w_down hold the same experts, [E, N, H] and [E, H, I]")
    weights, experts = route_experts(logits, top_k, **(routing or {}))
    plan = plan_dispatch(experts, w_up.shape[0])
    gate = {"slope": slope, "limit": limit, "shift": shift}
    caches = weight_caches or (None, None)
    params = (x, logits, w_up, w_down, bias_up, bias_down, residual)
    if (torch.is_grad_enabled() and main_grads is not None) or tracked(*params):
        mains, scales = main_grads or (None, None), scalings or (None, None)
        h = grouped_linear_fp8(dispatch_tokens(x, plan), w_up, plan.group_offs, mains[0], caches[0], scales[0],
                               bias=bias_up, activation=activation, **gate)
        y = grouped_linear_fp8(h, w_down, plan.group_offs, mains[1], caches[1], scales[1], bias=bias_down)
        return combine_tokens(y, plan, weights, residual)
    q, sx, _ = quantize_fp8_tensorwise(_rows16(x), "e4m3", slots=plan.slots)
    rows = dispatch_tokens(q, plan, row_align=_LINE)
    qu, su = _weight(w_up, caches[0])
    h = grouped_gemm_fp8_bias_act(rows, qu, sx, su, plan.group_offs, bias_up, activation, zero_tail=True, **gate)
    qh, sh, _ = quantize_fp8_tensorwise(h, "e4m3", row_align=_LINE)
    qd, sd = _weight(w_down, caches[1])
    y = grouped_gemm_fp8_bias_act(qh, qd, sh, sd, plan.group_offs, bias_down)
    return combine_tokens(y, plan, weights, residual)
