"""A whole MoE layer: routing, dispatch, the experts' two FP8 products and the combination.

``moe_layer_fp8`` is how the package's operators are meant to follow one another, ``moe_layer_mx`` the same on weights kept
in 4 bits; a model with another order of steps calls them one by one. The reference's harness runs the products alone, on
random rows (reference bench.py:196-268).
"""
from __future__ import annotations

import torch

from ._tensors import MXTensor, mx_columns, tracked
from .autograd import FP8DelayedScaling, FP8WeightCache, check_checkpoint, grouped_linear_fp8
from .moe import combine_tokens, dispatch_tokens, plan_dispatch, route_experts
from .mx import dispatch_mx, grouped_gemm_mx_bias_act, quantize_mx
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
                  scalings: tuple[FP8DelayedScaling, FP8DelayedScaling] | None = None,
                  checkpoint: str | None = None) -> torch.Tensor:
    """``residual + sum_j weight_j * expert_j(x)`` of every token, [T, H] bf16.

    x: bf16 [T, H]; logits: the router's, [T, E]; w_up: [E, N, H] and w_down: [E, H, I], bf16 / fp32, I = N / 2 for
    "swiglu" and N otherwise; biases [E, N] and [E, H]. ``routing``: options of ``route_experts``; ``slope``, ``limit``,
    ``shift``: of the activation; ``main_grads``, ``weight_caches``, ``scalings``: those of ``grouped_linear_fp8``, for
    the two products; ``checkpoint``: its, for the first one (nothing is kept without gradients).

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
    check_checkpoint(checkpoint)
    weights, experts = route_experts(logits, top_k, **(routing or {}))
    plan = plan_dispatch(experts, w_up.shape[0])
    gate = {"slope": slope, "limit": limit, "shift": shift}
    caches = weight_caches or (None, None)
    params = (x, logits, w_up, w_down, bias_up, bias_down, residual)
    if (torch.is_grad_enabled() and main_grads is not None) or tracked(*params):
        mains, scales = main_grads or (None, None), scalings or (None, None)
        h = grouped_linear_fp8(dispatch_tokens(x, plan), w_up, plan.group_offs, mains[0], caches[0], scales[0],
                               bias=bias_up, activation=activation, checkpoint=checkpoint, **gate)
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


def _copied_first(rows: int, features: int) -> bool:
    """Whether the copied rows are quantized, one launch fewer, or the tokens' blocks copied, a quarter (e2m1) or half of the
    bytes. The crossing lies at 2^25 values of the copied rows, whatever their features, top_k and format. Us so and by
    dispatch_mx, e4m3, top 4: 512 features 65536 rows 32 and 34, 131072 61 and 43; 2880 features 8192 rows 25 and 38, 16384 45 and
    39; 8192 features 4096 rows 33 and 34, 8192 62 and 34. Top 1: 65536 rows of 512 41 and 42, 4096 of 8192 40 and 36."""
    return rows * features <= 1 << 25


def moe_layer_mx(x: torch.Tensor, logits: torch.Tensor, w_up: MXTensor, w_down: MXTensor, top_k: int, *,
                 bias_up: torch.Tensor | None = None, bias_down: torch.Tensor | None = None,
                 activation: str | None = "swiglu", slope: float = 1.0, limit: float | None = None, shift: float = 0.0,
                 residual: torch.Tensor | None = None, routing: dict | None = None, fmt: str = "e4m3") -> torch.Tensor:
    """``residual + sum_j weight_j * expert_j(x)`` of every token, [T, H] bf16, for inference on microscaled weights.

    w_up, w_down: e2m1, the values of [E, N, H] and [E, H, I] (``quantize_mx(w, row_align=128)``; neighbouring rows of w_up
    are gate and value for "swiglu"); H and I multiples of 32. ``fmt``: what the activations are quantized to before each
    product, "e4m3" or "e2m1". The rest as for ``moe_layer_fp8``.

    A token's blocks are its own, so no scale is shared by a batch: a token's result does not depend on what it is batched
    with, but for the order of fp32 sums in another kernel. It has no gradients and refuses an input that asks for one."""
    if x.dim() != 2 or x.dtype != torch.bfloat16:
        raise TypeError("x must be a bf16 [T, H] tensor")
    if mx_columns(w_up, "w_up")[0] != 1 or mx_columns(w_down, "w_down")[0] != 1 or w_up.q.dim() != 3 or w_down.q.dim() != 3:
        raise TypeError("w_up and w_down must hold e2m1 values [E, N, H] and [E, H, I]")
    experts, hidden = w_up.q.shape[0], 2 * w_up.q.shape[2]
    if x.shape[1] != hidden:
        raise ValueError(f"x has {x.shape[1]} features, w_up {hidden}")
    if logits.dim() != 2 or logits.shape[0] != x.shape[0] or logits.shape[1] != experts:
        raise ValueError(f"logits must be [{x.shape[0]}, {experts}]")
    inner = w_up.q.shape[1] // (2 if activation == "swiglu" else 1)
    if tuple(w_down.q.shape) != (experts, hidden, inner // 2) or inner % 32:
        raise ValueError("w_up and w_down hold the same experts, [E, N, H] and [E, H, I], I a multiple of 32")
    if tracked(x, logits, bias_up, bias_down, residual):
        raise RuntimeError("moe_layer_mx has no gradients: call it under torch.no_grad()")
    weights, chosen = route_experts(logits, top_k, **(routing or {}))
    plan = plan_dispatch(chosen, experts)
    if _copied_first(plan.slots.numel(), hidden):
        rows = quantize_mx(dispatch_tokens(x, plan), fmt, _LINE)
    else:
        rows = dispatch_mx(quantize_mx(x, fmt), plan)
    h = grouped_gemm_mx_bias_act(rows, w_up, plan.group_offs, bias_up, activation, slope=slope, limit=limit, shift=shift)
    y = grouped_gemm_mx_bias_act(quantize_mx(h, fmt, _LINE), w_down, plan.group_offs, bias_down)
    return combine_tokens(y, plan, weights, residual)
