"""The MoE layer on 4-bit weights: its operators in a row against 64-bit arithmetic on the values that they hand each other,
its dispatch, a captured step, tokens that go nowhere, and what it refuses.
"""
import math

import pytest
import torch

from oracle import mx_oracle as omx
from test_gpu_mx import _check

pytestmark = pytest.mark.gpu

GATE = dict(slope=1.702, limit=7.0, shift=1.0)


def _layer(pkg, T, E, H, I, activation, seed, logits=None):
    gen = torch.Generator().manual_seed(seed)

    def make(*s, std=1.0):
        return (torch.randn(s, generator=gen) * std).to(torch.bfloat16).cuda()

    n = 2 * I if activation == "swiglu" else I
    x, wu, wd = make(T, H), make(E, n, H, std=H ** -0.5), make(E, H, I, std=I ** -0.5)
    bu, bd, res = make(E, n, std=0.2), make(E, H, std=0.2), make(T, H)
    logits = torch.randn((T, E), generator=gen).cuda() if logits is None else logits
    return x, logits, pkg.quantize_mx(wu, row_align=128), pkg.quantize_mx(wd, row_align=128), bu, bd, res


@pytest.mark.parametrize("T,E,k,H,I", [(1, 4, 2, 64, 32), (5, 8, 3, 160, 96), (77, 4, 4, 2880, 64), (700, 32, 4, 512, 736), (4200, 3, 2, 64, 64),
                                       (3000, 3, 2, 128, 2880)])
@pytest.mark.parametrize("activation,options", [("swiglu", GATE), ("swiglu", {}), ("gelu", {}), (None, {})])
@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_layer(pkg, T, E, k, H, I, activation, options, fmt):
    """Each product within its own bound of what 64 bits make of its operands; quantization and dispatch exact; the layer the
    same bits as its parts; the combination's k terms and the residual summed in fp32 and rounded once."""
    x, logits, wu, wd, bu, bd, res = _layer(pkg, T, E, H, I, activation, T + H)
    out = pkg.moe_layer_mx(x, logits, wu, wd, k, bias_up=bu, bias_down=bd, activation=activation, residual=res, fmt=fmt, **options)
    weights, chosen = pkg.route_experts(logits, k)
    plan = pkg.plan_dispatch(chosen, E)
    qx = pkg.quantize_mx(x, fmt)
    q, s = omx.quantize(x.cpu(), fmt)
    assert torch.equal(qx.q.cpu().view(torch.uint8), omx.store(q, fmt).view(torch.uint8)) and torch.equal(qx.scales.cpu(), s)
    rows = pkg.dispatch_mx(qx, plan)
    slots = plan.slots.long()
    for j in range(k):
        assert torch.equal(rows.q[slots[:, j]].view(torch.uint8), qx.q.view(torch.uint8))
        assert torch.equal(rows.scales[slots[:, j]], qx.scales)
    h = pkg.grouped_gemm_mx_bias_act(rows, wu, plan.group_offs, bu, activation, **options)
    qh = pkg.quantize_mx(h, fmt, 128)
    y = pkg.grouped_gemm_mx_bias_act(qh, wd, plan.group_offs, bd)
    assert torch.equal(out, pkg.combine_tokens(y, plan, weights, res))
    offs = plan.group_offs.tolist()

    def check(got, a, w, bias, act, **gate):
        # the bound of the product's own tests: the matrix cores' sums of e4m3 values, the activation's slope, one rounding
        z, ref, size = omx.product(omx.decode(a.q, a.scales), omx.decode(w.q, w.scales), fmt, offs, bias, act, None, **gate)
        _check(got.double(), z, ref, size, act, gate, torch.zeros_like(ref))

    check(h, rows, wu, bu, activation, **options)
    check(y, qh, wd, bd, None)


def test_a_token_alone_is_the_token_in_a_batch(pkg):
    """No scale is shared by a batch: the same rows come out, but for fp32 sums in another kernel's order."""
    x, logits, wu, wd, bu, bd, res = _layer(pkg, 300, 8, 256, 192, "swiglu", 1)
    args = dict(bias_up=bu, bias_down=bd, **GATE)
    out = pkg.moe_layer_mx(x, logits, wu, wd, 2, residual=res, **args)
    x[1:] *= 1e4
    again = pkg.moe_layer_mx(x, logits, wu, wd, 2, residual=res, **args)
    assert torch.equal(out[0], again[0])
    one = pkg.moe_layer_mx(x[:1], logits[:1], wu, wd, 2, residual=res[:1], **args)
    # h's values may round to neighbouring codes of e4m3 (2^-3 of a value, in a few of 192 terms)
    assert (one[0].float() - out[0].float()).norm() <= 0.02 * out[0].float().norm()


def test_masked_tokens_go_nowhere(pkg):
    x, logits, wu, wd, bu, bd, res = _layer(pkg, 40, 4, 64, 64, "swiglu", 2)
    logits[7], logits[39] = -math.inf, -math.inf
    x[7] = math.nan
    out = pkg.moe_layer_mx(x, logits, wu, wd, 2, bias_up=bu, bias_down=bd, residual=res)
    assert torch.equal(out[7], res[7]) and torch.equal(out[39], res[39]) and torch.isfinite(out).all()
    keep = [t for t in range(40) if t not in (7, 39)]
    assert torch.equal(out[keep], pkg.moe_layer_mx(x[keep], logits[keep], wu, wd, 2, bias_up=bu, bias_down=bd, residual=res[keep]))


def test_dispatch_of_views(pkg):
    """Rows of other strides, scales by blocks, buffers that end with the last scale."""
    gen = torch.Generator().manual_seed(3)
    for K in (32, 160, 528, 2880):
        for fmt in ("e4m3", "e2m1"):
            t = pkg.quantize_mx(torch.randn((30, K), generator=gen).cuda(), fmt)
            chosen = torch.randint(-1, 5, (30, 1), generator=gen, dtype=torch.int32).cuda()
            plan = pkg.plan_dispatch(chosen, 5)
            want = pkg.dispatch_mx(t, plan)
            tight = t.scales.clone(memory_format=torch.contiguous_format)
            exact = torch.empty(tight.numel(), dtype=torch.uint8, device="cuda").view(tight.shape).copy_(tight)
            for scales in (tight, exact, t.scales.t().contiguous().t()):
                for q in (t.q, t.q.view(torch.uint8).t().contiguous().t().view(t.q.dtype)):
                    got = pkg.dispatch_mx(pkg.MXTensor(q, scales), plan)
                    assert torch.equal(got.q.view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(got.scales, want.scales)
            end = int(plan.group_offs[-1])
            assert not want.q[end:].view(torch.uint8).any() and not want.scales[end:].any()
            assert want.q.stride(0) % 128 == 0 and want.scales.stride(0) % 16 == 0
    none = pkg.dispatch_mx(pkg.quantize_mx(torch.zeros((0, 64), device="cuda")), pkg.plan_dispatch(chosen[:0], 5))
    assert tuple(none.q.shape) == (0, 32) and tuple(none.scales.shape) == (0, 2)


def test_no_tokens(pkg):
    x, logits, wu, wd, bu, bd, res = _layer(pkg, 0, 4, 64, 64, "swiglu", 4)
    assert pkg.moe_layer_mx(x, logits, wu, wd, 2, bias_up=bu, residual=res).shape == (0, 64)


@pytest.mark.parametrize("T", [1, 300])
def test_captured(pkg, T):
    x, logits, wu, wd, bu, bd, res = _layer(pkg, T, 8, 128, 96, "swiglu", 5)

    def step():
        return pkg.moe_layer_mx(x, logits, wu, wd, 2, bias_up=bu, bias_down=bd, residual=res, **GATE)

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.synchronize()
    for _ in range(4):
        x.copy_(torch.randn(x.shape).to(torch.bfloat16))
        logits.copy_(torch.randn(logits.shape))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())


def test_refusals(pkg):
    x, logits, wu, wd, bu, bd, res = _layer(pkg, 6, 4, 64, 96, "swiglu", 6)
    e4 = pkg.quantize_mx(torch.zeros((4, 192, 64), device="cuda"), "e4m3")
    cases = [(TypeError, (x.float(), logits, wu, wd, 2), {}), (TypeError, (x, logits, e4, wd, 2), {}),
             (TypeError, (x, logits, wu, pkg.MXTensor(wd.q[0], wd.scales[0]), 2), {}),
             (ValueError, (x[:, :32], logits, wu, wd, 2), {}), (ValueError, (x, logits[:5], wu, wd, 2), {}),
             (ValueError, (x, logits[:, :3], wu, wd, 2), {}), (ValueError, (x, logits, wu, wd, 2), dict(activation="silu")),
             (ValueError, (x, logits, wu, pkg.MXTensor(wd.q[:3], wd.scales[:3]), 2), {}),
             (ValueError, (x, logits, wu, wd, 2), dict(fmt="e5m2")), (ValueError, (x, logits, wu, wd, 5), {}),
             (ValueError, (x, logits, wu, wd, 2), dict(bias_up=bu[:, :8])),
             (RuntimeError, (x.clone().requires_grad_(), logits, wu, wd, 2), {}),
             (RuntimeError, (x, logits, wu, wd, 2), dict(bias_down=bd.clone().requires_grad_()))]
    for exc, args, kw in cases:
        with pytest.raises(exc):
            pkg.moe_layer_mx(*args, **kw)
    with torch.no_grad():
        pkg.moe_layer_mx(x.clone().requires_grad_(), logits, wu, wd, 2)
    for bad in (pkg.MXTensor(wu.q, wu.scales), pkg.MXTensor(wu.q[0, :6], wu.scales[0, :6, :1])):
        with pytest.raises(ValueError):
            pkg.dispatch_mx(bad, pkg.plan_dispatch(torch.zeros((6, 1), dtype=torch.int32, device="cuda"), 4))


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_both_orders_of_copying_and_quantizing(pkg, fmt, monkeypatch):
    """Rows enough that the tokens' blocks are copied, tokens that go nowhere among them: the bits of the other order."""
    T, E, k, H = 3000, 8, 4, 2880
    logits = torch.randn((T, E), generator=torch.Generator().manual_seed(7))
    logits[1::97] = -math.inf
    x, logits, wu, wd, bu, bd, res = _layer(pkg, T, E, H, 64, "swiglu", 7, logits.cuda())
    x[1::97] = math.nan
    assert not pkg.layer._copied_first(T * k, H)

    def run():
        return pkg.moe_layer_mx(x, logits, wu, wd, k, bias_up=bu, bias_down=bd, residual=res, fmt=fmt, **GATE)

    out = run()
    assert torch.isfinite(out).all() and torch.equal(out[1::97], res[1::97])
    monkeypatch.setattr(pkg.layer, "_copied_first", lambda *_: True)
    assert torch.equal(out, run())
