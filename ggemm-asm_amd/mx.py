"""Microscaled (MX) rows as torch ops over the C ABI (include/ggemm_mx.h): blocks of 32 values along a row share a power
of two, the values are e2m1 (4 bits) or e4m3 (8 bits).

* ``quantize_mx`` / ``dequantize_mx``  -- rows to their blocks and back: weights in 4 bits, activation checkpoints in 8
* ``dispatch_mx``                      -- tokens' blocks into expert order
* ``grouped_gemm_mx_bias_act``         -- the grouped product of e2m1 weights with e2m1 or e4m3 activations, with bias,
  activation and residual in its epilogue

The training layer keeps the value before its activation so (``keep_preact="mxfp8"`` of ``grouped_gemm_fp8_bias_act``,
``checkpoint="mxfp8"`` of ``grouped_linear_fp8``).

``quantize_mxfp8_grouped`` makes its blocks along the token axis, for the weight gradient; these lie along the features,
the axis that the forward product sums over. The reference's products take per-tensor scales (reference
bench.py:238-247). Every launch goes through libggemm_vark.so on torch's current stream; there is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib
from ._tensors import MX_BLOCK as BLOCK, MXTensor, mx_columns, on_gpu as _on_gpu, row_stride as _stride, tracked
from .moe import DispatchPlan, dispatch_tokens
from .product import _act, _check_offs, _rows16
from .quant import _IN, _padded_empty
from .vark import _validate_offsets

_FORMATS = {"e4m3": 0, "e2m1": 1}
TILES = (0, 16, 32, 64, 128, 256)    # of ggemm_mx_product


def tile_rows(a_format: str, G: int, N: int, K: int, M: int, num_cus: int = 256) -> int:
    """Rows of the output tiles of the kernel that ``grouped_gemm_mx_bias_act`` runs on these sizes: 16, 32, 64,
    128 or 256."""
    return _lib.load().ggemm_mx_tile_rows(_FORMATS[a_format], G, N, K, M, num_cus)


# --------------------------------------------------------------------------- rows to blocks and back

def quantize_mx(x: torch.Tensor, fmt: str = "e2m1", row_align: int | None = None) -> MXTensor:
    """The rows of x (bf16 / fp32 [.., K], K a multiple of 16) in blocks of 32, the last one of a row 16 long where K is an
    odd multiple of 16.

    A block's exponent is the smallest at which its largest value, rounded as though the format had no largest one, stays
    within it: no value saturates by more than half a step. Values are rounded once, to nearest, ties to the even code. A
    block that holds an infinity or NaN has the scale 255 (NaN) and values 0. Values of 1.75 * 2^127 and more, which only
    fp32's and bf16's last binade holds, may come back as infinity.

    ``row_align=128`` starts the rows of q on 128-byte lines, as the grouped product reads them best; rows of scales start on
    multiples of 16 bytes (both are views of padded buffers, whose padding is not written). The result carries no graph."""
    if fmt not in _FORMATS:
        raise ValueError(f"fmt must be 'e2m1' or 'e4m3', got {fmt!r}")
    if x.dtype not in _IN:
        raise TypeError(f"x must be bfloat16 or float32, got {x.dtype}")
    if x.dim() < 2:
        raise ValueError("x must have at least 2 dimensions (rows x columns)")
    _on_gpu(x, "the quantizer")
    cols = x.shape[-1]
    if cols == 0 or cols % 16:
        raise ValueError(f"the last dimension must be a multiple of 16, got {cols}")
    x2 = x if x.dim() == 2 else x.reshape(-1, cols)
    if x2.stride(1) != 1 or x2.data_ptr() % 16 or x2.shape[0] > 1 and (x2.stride(0) * x2.element_size() % 16
                                                                       or x2.stride(0) < cols):
        x2 = x2.clone(memory_format=torch.contiguous_format)
    code, dev, rows = _FORMATS[fmt], x.device, x2.shape[0]
    dt, width = (torch.float8_e4m3fn, cols) if code == 0 else (torch.uint8, cols // 2)
    q = _padded_empty(x.shape[:-1] + (width,), row_align, dt, dev)
    blocks = -(-cols // BLOCK)
    pitch = -(-blocks // 16) * 16
    scales = x.new_empty(x.shape[:-1] + (pitch,), dtype=torch.uint8)
    if pitch != blocks:
        scales = scales.narrow(-1, 0, blocks)
    if rows:
        _lib.launch("ggemm_mx_quantize", dev, cols, x2.data_ptr(), _IN[x.dtype], rows, cols, _stride(x2), code, q.data_ptr(),
                    q.stride(-2) if rows > 1 else width, scales.data_ptr(), pitch)
    return MXTensor(q, scales)


def _even_rows(t: torch.Tensor, unit: int) -> torch.Tensor:
    """t as a 2-D tensor with contiguous rows that start on multiples of ``unit`` bytes (a copy where it is not)."""
    t2 = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    if t2.stride(1) != 1 or t2.data_ptr() % unit or t2.shape[0] > 1 and (t2.stride(0) % unit or t2.stride(0) < t2.shape[1]):
        return t2.clone(memory_format=torch.contiguous_format)
    return t2


def dequantize_mx(t: MXTensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that t stands for, bf16 or fp32 [.., K], contiguous. Exact: q times a power of two needs at most four
    bits, and both types hold its exponent but for the ends of bf16's range (below 2^-133 rounded). The result
    carries no graph."""
    if dtype not in _IN:
        raise TypeError(f"dtype must be bfloat16 or float32, got {dtype}")
    q, scales = t
    code, cols = mx_columns(t, "t")
    if q.dim() < 2:
        raise ValueError("t must have at least 2 dimensions (rows x columns)")
    _on_gpu(q, "the restoration")
    if cols == 0 or cols % 16:
        raise ValueError(f"the last dimension must stand for a multiple of 16 values, got {cols}")
    q2 = _even_rows(q, 4 if code else 8)
    s2 = scales if scales.dim() == 2 else scales.reshape(-1, scales.shape[-1])
    out = q.new_empty(q.shape[:-1] + (cols,), dtype=dtype)
    rows = q2.shape[0]
    if rows:
        _lib.launch("ggemm_mx_dequantize", q.device, cols, q2.data_ptr(), code, rows, cols, _stride(q2), s2.data_ptr(),
                    s2.stride(0), s2.stride(1), out.data_ptr(), _IN[dtype], cols)
    return out


# --------------------------------------------------------------------------- the product

def _padded(t: torch.Tensor, row: int) -> torch.Tensor:
    """t [.., n] copied to rows of ``row`` bytes on multiples of 16."""
    out = torch.empty(tuple(t.shape[:-1]) + (-(-row // 16) * 16,), dtype=torch.uint8, device=t.device)
    out[..., :t.shape[-1]] = t.view(torch.uint8)
    return out


def _product_rows(t: torch.Tensor, row: int, past: bool):
    """(tensor, row stride, group stride) of an operand's bytes or scales, of whose rows ``row`` bytes are read, more than
    they hold where ``past``: a copy where the rows are not contiguous, do not start on multiples of 16 bytes, overlap or end
    before that."""
    shape, strides = t.shape, t.stride()
    rows, rs = shape[-2], strides[-2]
    if rows == 1:
        rs = -(-row // 16) * 16
    last = (rows - 1) * rs + row                       # bytes of a group
    groups, gs = (shape[0], strides[0]) if len(shape) == 3 else (1, 0)
    if groups == 1:
        gs = -(-last // 16) * 16
    if (strides[-1] != 1 and shape[-1] > 1 or (t.data_ptr() | rs | gs) & 15 or rs < row or gs < last
            or past and t.storage_offset() + (groups - 1) * gs + last > t.untyped_storage().nbytes()):
        t = _padded(t, row)
        rs = t.stride(-2)
        gs = rows * rs
    return t, rs, gs


def dispatch_mx(t: MXTensor, plan: DispatchPlan) -> MXTensor:
    """The tokens' rows of t ([T, K]) in expert order, as ``dispatch_tokens`` copies them: [T * k, K], laid out as the grouped
    product reads them best. Rows of no expert are zero."""
    mx_columns(t, "t")
    q, scales = t
    if q.dim() != 2 or q.shape[1] == 0:
        raise ValueError("t must be a [T, K] tensor, K positive")
    _on_gpu(q, "the dispatch")
    blocks = scales.shape[1]
    row = -(-blocks // 16) * 16                                  # copied whole, 16 bytes at a time
    if q.shape[0]:
        scales, stride, _ = _product_rows(scales, row, row > blocks)
        scales = scales.as_strided((q.shape[0], row), (stride, 1))
    return MXTensor(dispatch_tokens(q, plan, row_align=128), dispatch_tokens(scales, plan, row_align=16)[:, :blocks])


def grouped_gemm_mx_bias_act(a: MXTensor, b: MXTensor, group_offs: torch.Tensor, bias: torch.Tensor | None = None,
                             activation: str | None = None, residual: torch.Tensor | None = None, *, slope: float = 1.0,
                             limit: float | None = None, shift: float = 0.0, zero_tail: bool = False,
                             validate: bool = False, tile: int = 0) -> torch.Tensor:
    """``out[r] = act(a[r] @ b[g]^T + bias[g]) + residual[r]`` for ``offs[g] <= r < offs[g+1]``: bf16, computed in fp32 and
    rounded once, of the values that a and b stand for.

    a: [M, K], e2m1 or e4m3; b: e2m1 [G, N, K] (stored as [G, N, K / 2] bytes); group_offs: int64 [G+1]; K a multiple of
    32, N of 16. Bias, activation, its options, residual, ``zero_tail`` and ``validate`` as for
    ``grouped_gemm_fp8_bias_act``. A block with the scale 255 makes the results that it reaches NaN.

    Operands as ``quantize_mx`` lays them out are read where they are. Others are copied at each call, unless rows of q
    and of scales start on multiples of 16 bytes and rows of scales can be read up to a multiple of 16: weights from
    elsewhere are laid out so once. ``tile``: rows of the output tiles (16, 32, 64, 128 or 256), 0 for the library's choice.
    An operator of inference: it has no gradients and refuses a bias or residual that asks for one."""
    code, K = mx_columns(a, "a")
    b_code, Kb = mx_columns(b, "b")
    if b_code != 1:
        raise TypeError("b must hold e2m1 values (uint8)")
    aq, bq = a.q, b.q
    if aq.dim() != 2 or bq.dim() != 3:
        raise ValueError("a must be 2-D [M, K] and b 3-D [G, N, K]")
    dev = aq.device
    _on_gpu(aq, "the product")
    group_offs = _check_offs(group_offs, dev)
    M, (G, N) = aq.shape[0], bq.shape[:2]
    if G != group_offs.numel() - 1:
        raise ValueError(f"b holds {G} groups, group_offs {group_offs.numel() - 1}")
    if Kb != K:
        raise ValueError(f"K of a ({K}) and b ({Kb}) differ")
    if K == 0 or K % BLOCK or N == 0 or N % 16:
        raise ValueError(f"K must be a multiple of {BLOCK} and N of 16, got {K} and {N}")
    if bq.device != dev:
        raise ValueError("all tensors must be on the same device")
    act, slope, limit, shift = _act(activation, slope, limit, shift)
    width = N // 2 if activation == "swiglu" else N
    if bias is not None and (bias.dtype not in _IN or tuple(bias.shape) != (G, N) or bias.device != dev):
        raise ValueError(f"bias must be bf16 or fp32 [{G}, {N}] on a's device")
    if residual is not None and (residual.dtype != torch.bfloat16 or tuple(residual.shape) != (M, width)
                                 or residual.device != dev):
        raise ValueError(f"residual must be bf16 [{M}, {width}] on a's device")
    if tile not in TILES:
        raise ValueError(f"tile must be one of {TILES}, got {tile}")
    if tracked(bias, residual):
        raise RuntimeError("grouped_gemm_mx_bias_act has no gradients: call it under torch.no_grad()")
    if validate:
        _validate_offsets(group_offs, M, mx=False)
    out = aq.new_empty((M, width), dtype=torch.bfloat16)
    if M == 0:
        return out
    if bias is not None:
        bias = bias.contiguous()
        if bias.data_ptr() % 16:
            bias = bias.clone()
    if residual is not None:
        residual = _rows16(residual)
    chunk = -(-K // 512) * 16
    past = chunk > K // BLOCK
    aq, sa, _ = _product_rows(aq, K // 2 if code else K, False)
    a_scales, sas, _ = _product_rows(a.scales, chunk, past)
    bq, sbn, sbg = _product_rows(bq, K // 2, False)
    b_scales, sbsn, sbsg = _product_rows(b.scales, chunk, past)
    sres = 0 if residual is None else _stride(residual)
    _lib.launch("ggemm_mx_product", dev, G | N | K | sa | sas | sbn | sbsn | sres, aq.data_ptr(), code, a_scales.data_ptr(),
                bq.data_ptr(), b_scales.data_ptr(), out.data_ptr(), None if bias is None else bias.data_ptr(),
                0 if bias is None else _IN[bias.dtype], None if residual is None else residual.data_ptr(),
                group_offs.data_ptr(), G, N, K, sa, sas, sbg, sbn, sbsg, sbsn, width, sres, act, slope, limit, shift, M,
                int(bool(zero_tail)), tile)
    return out
