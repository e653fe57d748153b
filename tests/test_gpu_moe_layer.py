"""The MoE layer's operators together: against the same layer in plain torch on the operands as quantized, and the
grouped linear layer's gradients through bias and activation."""
import os
import sys

import pytest
import torch

from conftest import ROOT
from oracle import product_oracle as orx

pytestmark = pytest.mark.gpu

GATE = dict(slope=1.702, limit=7.0, shift=1.0)


def _dequantized(pkg, t, fmt):
    q, s, _ = pkg.quantize_fp8_tensorwise(t.contiguous(), fmt)
    return q.cpu().double() * s.cpu().double()


@pytest.mark.parametrize("activation,options", [(None, {}), ("silu", {}), ("gelu", {}), ("swiglu", GATE)])
@pytest.mark.parametrize("bias_dtype", [torch.bfloat16, torch.float32])
def test_grouped_linear_with_bias_and_activation(pkg, activation, options, bias_dtype):
    """out, dx, dw and dbias in fp64 on the operands' quantized values: fp8 products carry bf16's rounding (2^-8) and
    their sums' error; 2e-2 of the largest value is the products' parity bar."""
    gen = torch.Generator().manual_seed(3)
    lens, K, N = [40, 0, 1, 87], 160, 96
    M, G = sum(lens) + 6, len(lens)
    offs = [0]
    for n in lens:
        offs.append(offs[-1] + n)
    x = torch.randn((M, K), generator=gen).to(torch.bfloat16).cuda().requires_grad_()
    w = (torch.randn((G, N, K), generator=gen) * 0.1).to(torch.bfloat16).cuda().requires_grad_()
    b = torch.randn((G, N), generator=gen).to(bias_dtype).cuda().requires_grad_()
    width = N // 2 if activation == "swiglu" else N
    dout = torch.randn((M, width), generator=gen).to(torch.bfloat16).cuda()
    out = pkg.grouped_linear_fp8(x, w, torch.tensor(offs).cuda(), bias=b, activation=activation, **options)
    assert tuple(out.shape) == (M, width) and not out[offs[-1]:].any()
    out.backward(dout)
    xq, wq = _dequantized(pkg, x.detach(), "e4m3"), _dequantized(pkg, w.detach(), "e4m3")
    z = torch.zeros((M, N), dtype=torch.float64)
    for g in range(G):
        lo, hi = offs[g], offs[g + 1]
        z[lo:hi] = xq[lo:hi] @ wq[g].t() + b[g].detach().cpu().double()
    ref = orx.act(z, activation, **options)
    ref[offs[-1]:] = 0

    def near(got, want):
        assert (got.detach().cpu().double() - want).abs().max() <= 2e-2 * want.abs().max()

    near(out, ref)
    pre = z.to(torch.bfloat16)
    dz, dbias, _ = orx.backward(dout.cpu(), pre, offs, activation, **options)
    near(b.grad, dbias)
    assert b.grad.dtype == bias_dtype
    dq = _dequantized(pkg, dz.to(torch.bfloat16).cuda(), "e5m2")
    dx, dw = torch.zeros((M, K), dtype=torch.float64), torch.zeros((G, N, K), dtype=torch.float64)
    for g in range(G):
        lo, hi = offs[g], offs[g + 1]
        dx[lo:hi], dw[g] = dq[lo:hi] @ wq[g], dq[lo:hi].t() @ xq[lo:hi]
    # a dz one bf16 step away can round to the next e5m2 value, 2^-2 of it: in sums over N or the rows
    for got, want in ((x.grad, dx), (w.grad, dw)):
        err = (got.detach().cpu().double() - want).norm() / want.norm()
        assert err <= 2e-2, err


def test_without_bias_and_activation_the_layer_is_as_it_was(pkg):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn((50, 64), generator=gen).to(torch.bfloat16).cuda()
    w = torch.randn((2, 48, 64), generator=gen).to(torch.bfloat16).cuda()
    offs = torch.tensor([0, 20, 50]).cuda()
    qx, sx, _ = pkg.quantize_fp8_tensorwise(x, "e4m3", row_align=128)
    qw, sw, _ = pkg.quantize_fp8_tensorwise(w, "e4m3", row_align=128)
    assert torch.equal(pkg.grouped_linear_fp8(x, w, offs), pkg.grouped_gemm_fp8_tensorwise(qx, qw, sx, sw, offs))


@pytest.mark.parametrize("T", [1, 77])
def test_layer_with_and_without_gradients(pkg, T):
    """The training path's output, its gradients all there, against the inference path (the same products on the same
    quantized values, as every token is dispatched) and plain torch in fp32 on bf16 weights (fp8's 2^-4 per operand
    value: 0.1 of the norm)."""
    gen = torch.Generator().manual_seed(T)
    E, k, H, I = 8, 3, 128, 96

    def make(*s, std=1.0):
        return (torch.randn(s, generator=gen) * std).to(torch.bfloat16).cuda().requires_grad_()

    x, logits = make(T, H), make(T, E)
    wu, bu, wd, bd = make(E, 2 * I, H, std=0.1), make(E, 2 * I, std=0.1), make(E, H, I, std=0.1), make(E, H, std=0.1)
    args = dict(bias_up=bu, bias_down=bd, residual=x, routing=dict(score="sigmoid", scale=2.0), **GATE)
    out = pkg.moe_layer_fp8(x, logits, wu, wd, k, **args)
    out.float().square().mean().backward()
    for t in (x, logits, wu, bu, wd, bd):
        assert t.grad is not None and torch.isfinite(t.grad).all() and t.grad.any()
    with torch.no_grad():
        again = pkg.moe_layer_fp8(x, logits, wu, wd, k, **args)
        p = torch.sigmoid(logits.float())
        top = p.topk(k, 1)
        ref = x.float().clone()
        for j in range(k):
            e = top.indices[:, j]
            z = torch.bmm(wu[e].float(), x.float()[:, :, None])[:, :, 0] + bu[e].float()
            h = orx.act(z.double(), "swiglu", **GATE).float()
            y = torch.bmm(wd[e].float(), h[:, :, None])[:, :, 0] + bd[e].float()
            ref += y * (2.0 * top.values[:, j] / top.values.sum(1))[:, None]
    assert torch.equal(out, again)
    assert (out.float() - ref).norm() <= 0.1 * (ref - x.float()).norm()


def test_layer_refusals(pkg):
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    logits, w = torch.zeros((4, 2), device="cuda"), torch.zeros((2, 64, 64), device="cuda")
    for exc, f in [(TypeError, lambda: pkg.moe_layer_fp8(x.float(), logits, w, w, 1)),
                   (ValueError, lambda: pkg.moe_layer_fp8(x, logits[:3], w, w, 1)),
                   (ValueError, lambda: pkg.moe_layer_fp8(x, logits, w, w[:1], 1)),
                   (ValueError, lambda: pkg.grouped_linear_fp8(x, w, torch.tensor([0, 1, 4]).cuda(), activation="tanh"))]:
        with pytest.raises(exc):
            f()


def test_example_trains(pkg, monkeypatch):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import moe_layer
    monkeypatch.setattr(sys, "argv", ["moe_layer.py", "--tokens", "200", "--experts", "4", "--top-k", "2", "--hidden", "128",
                                      "--inner", "64", "--steps", "4"])
    losses = moe_layer.main()
    assert losses[-1] < losses[0]


@pytest.mark.parametrize("hidden,inner", [(144, 64), (64, 144), (160, 96)])
def test_example_runs_at_any_size_of_the_layer(pkg, monkeypatch, capsys, hidden, inner):
    """Multiples of 16 that are none of 32 too, which 4-bit weights do not take."""
    monkeypatch.syspath_prepend(os.path.join(ROOT, "examples"))
    import moe_layer
    monkeypatch.setattr(sys, "argv", ["moe_layer.py", "--tokens", "50", "--experts", "4", "--top-k", "2", "--hidden", str(hidden),
                                      "--inner", str(inner), "--steps", "1"])
    moe_layer.main()
    assert ("weights in 4 bits, " in capsys.readouterr().out) == (hidden % 32 == inner % 32 == 0)
