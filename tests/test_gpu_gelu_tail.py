"""gelu and its gradient where the normal distribution's cdf is small, in fp32 and against the tail's own size.

Tolerances, of units 2^-23. gauss(z) = e^(-z^2 / 2) by an exp2 whose argument, z^2 / 2 log2 e at most, carries two
roundings: z^2 units cover them. The rest of the cdf is a reciprocal, a polynomial and a few products: 16. The gradient cdf + z
pdf is held to its two terms' sizes, within 8 + z^2 units (its own factors are fewer). bf16 results are what values
within those units round to: for nearly every z one number.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -23


def _cdf(z):
    return 0.5 * torch.erfc(-z * math.sqrt(0.5))


# rows and features that take the kernels of 16, 64, 128 and 192 rows
@pytest.mark.parametrize("M,N,G,rows", [(2, 5760, 1, 16), (64, 1024, 1, 64), (3000, 2048, 1, 128), (20000, 2096, 1, 192)])
def test_gelu_far_below_zero_is_as_exact_as_near_it(pkg, M, N, G, rows):
    """z is the bias alone (zero operands), from -12.5 to 6."""
    from ggemm_asm_amd import product
    K = {16: 2064, 192: 2880}.get(rows, 128)
    assert product.tile_rows(G, N, K, M, "gelu") == rows
    bias = torch.linspace(-12.5, 6.0, N)[None].contiguous()
    a = torch.zeros((M, K), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    b = torch.zeros((G, N, K), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    one = torch.ones((), device="cuda")
    out = pkg.grouped_gemm_fp8_bias_act(a, b, one, one, torch.tensor([0, M]).cuda(), bias.cuda(), "gelu")
    z = bias[0].double()
    want = z * _cdf(z)
    assert (out == out[0]).all()
    off = (16 + z * z) * U * want.abs()
    got, least, most = out[0].cpu().float(), (want - off).to(torch.bfloat16).float(), (want + off).to(torch.bfloat16).float()
    assert ((least <= got) & (got <= most)).all(), ((got - want) / want).abs().max()
    assert (least == most).double().mean() > 0.99


def test_gelu_gradient_within_fp32(pkg):
    """One row a group, so that the bias' gradient is the factor in fp32."""
    z = torch.cat((torch.linspace(-12.5, 6.0, 4000), torch.linspace(-2, 2, 96))).to(torch.bfloat16)
    pre = z.view(2, 2048).cuda()
    _, dbias = pkg.bias_act_backward(torch.ones_like(pre), pre, torch.tensor([0, 1, 2]).cuda(), "gelu")
    v = z.double()
    cdf, pdf = _cdf(v), torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    err = (dbias.cpu().double().flatten() - (cdf + v * pdf)).abs()
    assert (err <= (8 + v * v) * U * (cdf + v.abs() * pdf) + 1e-37).all(), err.max()
