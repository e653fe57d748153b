"""The grouped FP8 product with bias, activation and residual in its epilogue, and the gradient of bias and activation,
as torch ops over the C ABI (include/ggemm_product.h).

``grouped_gemm_fp8_bias_act`` is ``grouped_gemm_fp8_tensorwise`` with what an expert's layer does next applied to the
fp32 accumulators, so that the wide result need not go to memory and back; ``bias_act_backward`` is its counterpart
before the data and weight gradients' products. The reference's products end at the scaled bf16 result (reference
bench.py:238-247). Every launch goes through libggemm_vark.so on torch's current stream; there is no CPU path.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from ._tensors import MX_BLOCK, MXTensor, mx_columns, on_gpu as _on_gpu, once_differentiable, row_stride as _stride, tracked
from .vark import _validate_offsets

MX8 = "mxfp8"            # of keep_preact: e4m3 in blocks of 32 columns
ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "swiglu": 3}
_IN = {torch.bfloat16: 0, torch.float32: 1}
MAX_GROUPS = 2047


def _act(activation, slope, limit, shift):
    """(code, slope, limit, shift) of an activation and its options."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be None, 'silu', 'gelu' or 'swiglu', got {activation!r}")
    if activation != "swiglu" and (slope != 1.0 or limit is not None or shift != 0.0):
        raise ValueError("slope, limit and shift are options of 'swiglu'")
    if limit is not None and not limit > 0:
        raise ValueError(f"limit must be positive, got {limit}")
    return ACTIVATIONS[activation], float(slope), float("inf") if limit is None else float(limit), float(shift)


def tile_rows(G: int, N: int, K: int, M: int, activation: str | None = None, *, keep_preact: bool = False,
              residual: bool = False, num_cus: int = 256) -> int:
    """Rows of the output tiles of the kernel that ``grouped_gemm_fp8_bias_act`` runs on contiguous tensors of these
    sizes: 16 (few rows), 64 or 128 (mid tiles), 192 (512 threads) or 256 (wide tiles)."""
    return _lib.load().ggemm_product_tile_rows(G, N, K, K, K, N // 2 if activation == "swiglu" else N,
                                               N if keep_preact else 0, ACTIVATIONS[activation], int(residual), M, num_cus)


def _check_offs(group_offs, dev):
    """The offsets as the kernels read them, one behind the other (a copy where they are not)."""
    if group_offs.dtype != torch.int64 or group_offs.dim() != 1 or not 2 <= group_offs.numel() <= MAX_GROUPS + 1:
        raise ValueError(f"group_offs must be int64 [G+1] with G <= {MAX_GROUPS}")
    if group_offs.device != dev:
        raise ValueError("all tensors must be on the same device")
    return group_offs.contiguous()


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """A 2-D bf16 tensor whose rows the kernels can read 16 bytes at a time (a copy where they cannot)."""
    if t.stride(1) != 1 or t.data_ptr() % 16 or t.shape[0] > 1 and (t.stride(0) % 8 or t.stride(0) < t.shape[1]):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _product(bias, residual, keep, a, b, a_scale, b_scale, group_offs, M, N, K, G, width, dev, code, slope, limit, shift,
             zero_tail):
    """(out, preact or None) of checked arguments."""
    if bias is not None:
        bias = bias.detach().contiguous()
        if bias.data_ptr() % 16:
            bias = bias.clone()
    if residual is not None:
        residual = _rows16(residual)
    out = torch.empty((M, width), dtype=torch.bfloat16, device=dev)
    if keep == MX8:
        # a row's scales lie apart: the kernels hold a block's scales of neighbouring rows
        by_block = torch.empty((-(-N // MX_BLOCK), -(-M // 16) * 16), dtype=torch.uint8, device=dev)
        pre = MXTensor(torch.empty((M, N), dtype=torch.float8_e4m3fn, device=dev), by_block.t()[:M])
    else:
        pre = torch.empty((M, N), dtype=torch.bfloat16, device=dev) if keep else None
    if M:
        # the strides of dimensions of size one are arbitrary and not used
        sam, sbn = a.stride(0) if M > 1 else K, b.stride(1)
        sbg = b.stride(0) if G > 1 else N * sbn
        sres = 0 if residual is None else _stride(residual)
        if keep == MX8:
            _lib.launch("ggemm_mx_keep_product", dev, G | N | K | sam | sbg | sbn | sres, a.data_ptr(), b.data_ptr(),
                        out.data_ptr(), pre.q.data_ptr(), by_block.data_ptr(), a_scale.data_ptr(), b_scale.data_ptr(),
                        None if bias is None else bias.data_ptr(), 0 if bias is None else _IN[bias.dtype],
                        None if residual is None else residual.data_ptr(), group_offs.data_ptr(), G, N, K, sam, sbg, sbn,
                        width, N, by_block.shape[1], sres, code, slope, limit, shift, M, int(bool(zero_tail)))
            return out, pre
        _lib.launch("ggemm_product_fp8_bias_act", dev, G | N | K | sam | sbg | sbn | sres, a.data_ptr(), b.data_ptr(),
                    out.data_ptr(), None if pre is None else pre.data_ptr(), a_scale.data_ptr(), b_scale.data_ptr(),
                    None if bias is None else bias.data_ptr(), 0 if bias is None else _IN[bias.dtype],
                    None if residual is None else residual.data_ptr(), group_offs.data_ptr(), G, N, K, sam, sbg, sbn,
                    width, N, sres, code, slope, limit, shift, M, int(bool(zero_tail)))
    return out, pre


def _kept(parts):
    """What _product kept, of its tensors."""
    return MXTensor(*parts) if len(parts) == 2 else parts[0]


class _BiasAct(torch.autograd.Function):
    """The product as a function of its bias and residual: the fp8 operands have no gradients."""

    @staticmethod
    def forward(ctx, bias, residual, keep_preact, group_offs, activation, options, args):
        for_bias = activation is not None and ctx.needs_input_grad[0]     # its gradient reads z
        out, pre = _product(bias, residual, keep_preact or for_bias, *args)
        parts = pre if isinstance(pre, MXTensor) else (pre,)
        ctx.save_for_backward(group_offs, *(parts if for_bias else ()))
        ctx.activation, ctx.options = activation, options
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        if not keep_preact:
            return out
        ctx.mark_non_differentiable(*parts)
        return (out, *parts)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, *_):
        group_offs, *parts = ctx.saved_tensors
        dbias = dres = None
        if dout is not None and ctx.needs_input_grad[0]:
            pre = _kept(parts) if parts else None
            _, dbias = bias_act_backward(dout, pre, group_offs, ctx.activation, **ctx.options)
            dbias = dbias.to(ctx.bias_dtype)
        if dout is not None and ctx.needs_input_grad[1]:
            # rows of no group are not written: they are no function of the residual
            row = torch.arange(dout.shape[0], device=dout.device)
            dres = torch.where(((row >= group_offs[0]) & (row < group_offs[-1]))[:, None], dout, 0)
        return dbias, dres, None, None, None, None, None


def grouped_gemm_fp8_bias_act(a: torch.Tensor, b: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor,
                              group_offs: torch.Tensor, bias: torch.Tensor | None = None,
                              activation: str | None = None, residual: torch.Tensor | None = None, *,
                              slope: float = 1.0, limit: float | None = None, shift: float = 0.0,
                              keep_preact: bool | str = False, zero_tail: bool = False, validate: bool = False):
    """``out[r] = act(a_scale * b_scale * a[r] @ b[g]^T + bias[g]) + residual[r]`` for ``offs[g] <= r < offs[g+1]``: bf16,
    computed in fp32 and rounded once.

    a: float8_e4m3fn [M, K]; b: float8_e4m3fn [G, N, K]; scales: single-element fp32 tensors; group_offs: int64 [G+1];
    K and N multiples of 16 (as ``grouped_gemm_fp8_tensorwise``). bias: bf16 or fp32 [G, N]. ``activation``: None,
    "silu", "gelu" (by the error function) or "swiglu" over pairs of columns z[:, 2i], z[:, 2i + 1]:
    ``g / (1 + exp(-slope * g)) * (u + shift)`` with ``g = min(z[:, 2i], limit)`` and ``u`` the other clamped to
    +-limit, which halves the width. residual: bf16, as wide as the result. With ``keep_preact`` the result is
    ``(out, preact)``, preact the bf16 [M, N] value before the activation, for ``bias_act_backward``; with
    ``keep_preact="mxfp8"`` preact is an ``MXTensor``, the same in 8 bits and a scale for 32 columns, quantized from fp32
    (an activation is needed: without one preact is the result). Rows outside
    ``[0, offs[G])`` are left unwritten, or zero from offs[G] on with ``zero_tail``. ``validate=True`` checks group_offs
    on the host first (a sync).

    Differentiable by bias and residual (``grouped_linear_fp8`` is by the activations and weights too); the value before
    the activation is then kept for the bias' gradient, in 8 bits with ``keep_preact="mxfp8"``, else in bf16, and the
    gradient is taken at what is kept. A ``preact`` that is returned carries no gradient itself."""
    if a.dim() != 2 or b.dim() != 3:
        raise ValueError("a must be 2-D [M, K] and b 3-D [G, N, K]")
    if a.dtype != torch.float8_e4m3fn or b.dtype != torch.float8_e4m3fn:
        raise TypeError(f"a and b must be float8_e4m3fn, got {a.dtype} and {b.dtype}")
    dev = a.device
    _on_gpu(a, "the product")
    group_offs = _check_offs(group_offs, dev)
    (M, K), (G, N, Kb) = a.shape, b.shape
    if G != group_offs.numel() - 1:
        raise ValueError(f"b holds {G} groups, group_offs {group_offs.numel() - 1}")
    if Kb != K:
        raise ValueError(f"K of a ({K}) and b ({Kb}) differ")
    if a.stride(1) != 1 or b.stride(2) != 1:
        raise ValueError("a and b must be contiguous along K")
    for s in (a_scale, b_scale):
        if s.dtype != torch.float32 or s.numel() != 1 or s.device != dev:
            raise ValueError("scales must be single-element fp32 tensors on a's device")
    if b.device != dev:
        raise ValueError("all tensors must be on the same device")
    code, slope, limit, shift = _act(activation, slope, limit, shift)
    if isinstance(keep_preact, str):
        if keep_preact != MX8:
            raise ValueError(f"keep_preact must be a bool or {MX8!r}, got {keep_preact!r}")
        if activation is None:
            raise ValueError(f"keep_preact={MX8!r} needs an activation: without one the value before it is the result")
    width = N // 2 if activation == "swiglu" else N
    if bias is not None:
        if bias.dtype not in _IN or tuple(bias.shape) != (G, N) or bias.device != dev:
            raise ValueError(f"bias must be bf16 or fp32 [{G}, {N}] on a's device")
    if residual is not None:
        if residual.dtype != torch.bfloat16 or tuple(residual.shape) != (M, width) or residual.device != dev:
            raise ValueError(f"residual must be bf16 [{M}, {width}] on a's device")
    if validate:
        _validate_offsets(group_offs, M, mx=False)
    if tracked(bias, residual):
        options = {"slope": slope, "limit": limit, "shift": shift} if activation == "swiglu" else {}
        got = _BiasAct.apply(bias, residual, keep_preact, group_offs, activation, options,
                             (a, b, a_scale, b_scale, group_offs, M, N, K, G, width, dev, code, slope, limit, shift, zero_tail))
        return (got[0], _kept(got[1:])) if keep_preact else got
    out, pre = _product(bias, residual, keep_preact, a, b, a_scale, b_scale, group_offs, M, N, K, G, width, dev, code, slope,
                        limit, shift, zero_tail)
    return (out, pre) if keep_preact else out


def _kept_rows(preact: MXTensor, M: int, N: int, dev):
    """An 8-bit checkpoint of [M, N] values whose rows the gradient's kernel can read 8 bytes at a time."""
    code, cols = mx_columns(preact, "preact")
    if code != 0 or tuple(preact.q.shape) != (M, N) or preact.q.device != dev:
        raise ValueError(f"preact must hold float8_e4m3fn [{M}, {N}] on dout's device")
    q = preact.q
    if q.stride(1) != 1 or q.data_ptr() % 8 or M > 1 and (q.stride(0) % 8 or q.stride(0) < N):
        q = q.clone(memory_format=torch.contiguous_format)
    return q, preact.scales


@functools.lru_cache(maxsize=256)                    # a size, no memory: the call is a twelfth of the whole one's time
def _workspace(mx: bool, M: int, G: int, N: int) -> int:
    lib = _lib.load()
    return (lib.ggemm_mx_act_workspace if mx else lib.ggemm_product_act_workspace)(M, G, N)


def bias_act_backward(dout: torch.Tensor, preact: torch.Tensor | MXTensor | None, group_offs: torch.Tensor,
                      activation: str | None = None, *, slope: float = 1.0, limit: float | None = None,
                      shift: float = 0.0, bias_grad: bool = True):
    """``(dpreact, dbias)`` of ``act(preact)`` and its bias: dpreact bf16 [M, N] = dout * act'(preact), dbias fp32 [G, N]
    the sum of it over each group's rows before its rounding (None without ``bias_grad``). Rows outside the groups are
    in no sum and get zero gradient.

    dout: bf16 [M, N] ([M, N / 2] for "swiglu"); preact: what ``grouped_gemm_fp8_bias_act`` kept, bf16 or (an
    ``MXTensor``) 8-bit: the gradient is that of the kept values; without an activation
    it may be None, and dpreact is dout itself, all its rows. Sums are made in a fixed order: the same inputs give the
    same bits. The results carry no graph."""
    code, slope, limit, shift = _act(activation, slope, limit, shift)
    if dout.dim() != 2 or dout.dtype != torch.bfloat16:
        raise TypeError("dout must be a bf16 [M, N] tensor")
    dev = dout.device
    _on_gpu(dout, "the gradient")
    group_offs = _check_offs(group_offs, dev)
    M = dout.shape[0]
    N = dout.shape[1] * (2 if activation == "swiglu" else 1)
    if N % 16 or N == 0:
        raise ValueError(f"N must be a multiple of 16, got {N}")
    kept = None
    if activation is not None and isinstance(preact, MXTensor):
        kept = _kept_rows(preact, M, N, dev)
        dpre = dout.new_empty((M, N))
    elif activation is not None:
        if preact is None or preact.dtype != torch.bfloat16 or tuple(preact.shape) != (M, N) or preact.device != dev:
            raise ValueError(f"preact must be bf16 [{M}, {N}] on dout's device")
        preact = _rows16(preact)
        dpre = torch.empty((M, N), dtype=torch.bfloat16, device=dev)
    else:
        preact, dpre = None, None
    G = group_offs.numel() - 1
    src = _rows16(dout)
    dbias = dout.new_empty((G, N), dtype=torch.float32) if bias_grad else None
    if M and (bias_grad or dpre is not None):
        ws = dout.new_empty(_workspace(kept is not None, M, G, N), dtype=torch.float32) if bias_grad else None
        if kept is not None:
            q, scales = kept
            _lib.launch("ggemm_mx_act_backward", dev, G | N | _stride(src) | _stride(q), src.data_ptr(), q.data_ptr(),
                        scales.data_ptr(), group_offs.data_ptr(), G, N, _stride(src), _stride(q), scales.stride(0),
                        scales.stride(1), code, slope, limit, shift, M, dpre.data_ptr(), N,
                        None if dbias is None else dbias.data_ptr(), None if ws is None else ws.data_ptr())
            return dpre, dbias
        spre = 0 if preact is None else _stride(preact)
        _lib.launch("ggemm_product_act_backward", dev, G | N | _stride(src) | spre, src.data_ptr(),
                    None if preact is None else preact.data_ptr(), group_offs.data_ptr(), G, N, _stride(src), spre, code,
                    slope, limit, shift, M, None if dpre is None else dpre.data_ptr(), N,
                    None if dbias is None else dbias.data_ptr(), None if ws is None else ws.data_ptr())
    elif dbias is not None:
        dbias.zero_()
    return dout if dpre is None else dpre, dbias
