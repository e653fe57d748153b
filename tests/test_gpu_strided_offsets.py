"""Group offsets that lie apart in memory, as a column of a table does: every operator that takes offsets gives the bits that
the same offsets one behind the other give. What lies between them is a repetition, so that either way of reading is in range.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

OFFS = [0, 70, 70, 200, 290]
M, K, N, G = 300, 128, 320, 4


@pytest.fixture(scope="module")
def offsets():
    tight = torch.tensor(OFFS).cuda()
    return tight, tight.repeat_interleave(2).view(-1, 2)[:, 0]


@pytest.fixture(scope="module")
def operands():
    gen = torch.Generator().manual_seed(1)
    a, b = (torch.randn(s, generator=gen).to(torch.float8_e4m3fn).cuda() for s in ((M, K), (G, N, K)))
    one = torch.ones((), device="cuda")
    bias = torch.randn((G, N), generator=gen).cuda()
    dout = torch.randn((M, N), generator=gen).to(torch.bfloat16).cuda()
    return a, b, one, bias, dout


def _same(got, want):
    got, want = ([t if isinstance(t, tuple) else (t,) for t in r] for r in (got, want))
    for g, w in zip(got, want):
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(g, w))


def test_products_with_an_epilogue(pkg, offsets, operands):
    a, b, one, bias, dout = operands

    def run(offs):
        out, pre = pkg.grouped_gemm_fp8_bias_act(a, b, one, one, offs, bias, "silu", keep_preact=True, zero_tail=True)
        also, kept = pkg.grouped_gemm_fp8_bias_act(a, b, one, one, offs, bias, "silu", keep_preact="mxfp8", zero_tail=True)
        return (out, pre, also, kept.q, kept.scales.contiguous(), pkg.bias_act_backward(dout, pre, offs, "silu"),
                pkg.bias_act_backward(dout, kept, offs, "silu"), pkg.bias_act_backward(dout, None, offs))

    _same(*map(run, reversed(offsets)))


def test_products_and_weight_gradients(pkg, offsets, operands):
    from ggemm_asm_amd.vark import weight_grad_fp8
    a, b, one, _, dout = operands
    dy = dout.to(torch.float8_e5m2)

    def run(offs):
        x = torch.randn((M, K), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
        (q, scales, padded), (qd, sd, _) = pkg.quantize_mxfp8_grouped(x, offs), pkg.quantize_mxfp8_grouped(dout, offs, "e5m2")
        end = int(padded[-1])
        return (pkg.grouped_gemm_fp8_tensorwise(a, b, one, one, offs, zero_tail=True), weight_grad_fp8(dy, a, one, one, offs),
                pkg.grouped_gemm_fp8_tensorwise_variable_k(a, dy, one, one, offs), q[:end], scales[:end // 32], padded,
                pkg.grouped_gemm_mxfp8_variable_k(q, qd, scales, sd, padded),
                pkg.grouped_gemm_mxfp8_variable_k(q, qd, scales, sd, padded.repeat_interleave(2).view(-1, 2)[:, 0]))

    got, want = map(run, reversed(offsets))
    _same(got, want)
    _same(got[-2:-1], got[-1:])


def test_layers(pkg, offsets, operands):
    gen = torch.Generator().manual_seed(3)
    x, w = torch.randn((M, K), generator=gen).to(torch.bfloat16).cuda(), torch.randn((G, N, K), generator=gen).to(torch.bfloat16).cuda()
    bias, dout = operands[3:]

    def run(offs, **options):
        leaves = [t.clone().requires_grad_() for t in (x, w, bias)]
        out = pkg.grouped_linear_fp8(leaves[0], leaves[1], offs, bias=leaves[2], activation="gelu", **options)
        out.backward(dout)
        return (out.detach(), *(t.grad for t in leaves))

    for options in ({}, {"checkpoint": "mxfp8"}):
        _same(*(run(offs, **options) for offs in reversed(offsets)))
    weights = pkg.quantize_mx(w, row_align=128)
    rows = pkg.quantize_mx(x, "e4m3", 128)
    _same(*([pkg.grouped_gemm_mx_bias_act(rows, weights, offs, bias, zero_tail=True)] for offs in reversed(offsets)))
