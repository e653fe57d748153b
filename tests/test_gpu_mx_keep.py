"""The value before an activation kept in 8 bits, on the GPU: the product that keeps it against the 64-bit oracle, the gradient
from it against the oracle and, bit for bit, against the bf16 path, and the layers that use both.

Tolerances. Kept values: z has the error of the matrix cores' fp8 sums (``product_oracle.product``'s bound d); a value kept
with exponent X is its z rounded to e4m3: off by 2^-4 of it, or 2^-10 2^X below the format's normal numbers. X is the
oracle's for a block maximum within the bound. What is kept is exact in bf16, so the gradient from it has to be that of the
restored bf16 tensor, bit for bit. The bias' sums add the same terms x in the same order, but a compiler may round a term
before it adds it or with it: a term is off by 2^-24 of it, either sum of n terms by n 2^-24 of the sum of |x|, and |x| is
known from bf16's rounding of it (1 + 2^-8).
"""
import math

import pytest
import torch

from oracle import mx_oracle as omx, product_oracle as orx
from test_gpu_product import GATE, KERNELS, SHAPES, _check, _inputs, _strided

pytestmark = pytest.mark.gpu

BF = 2.0 ** -8
ACTS = [("silu", {}), ("gelu", {}), ("swiglu", {}), ("swiglu", GATE)]


def _check_kept(kept, z, size):
    """Kept values and exponents of the rows that z has (NaN elsewhere), against z and its bound."""
    live = ~torch.isnan(z).any(1)
    q, scales, z, d = kept.q[live], kept.scales[live], z[live], size[live]
    got = omx.decode(q, scales)
    X = scales.double() - 127
    power = torch.exp2(X).repeat_interleave(32, 1)[:, :z.shape[1]]
    bad = ~((got - z).abs() <= d + 2.0 ** -4 * (z.abs() + d) + 2.0 ** -10 * power)
    assert not bad.any(), ((got - z).abs()[bad].max(), bad.nonzero()[:4])
    pad = -z.shape[1] % 32

    def exponents(v):                              # as the oracle's rule, of block maxima
        top = torch.nn.functional.pad(v, (0, pad)).view(v.shape[0], -1, 32).amax(2)
        x = torch.floor(torch.log2(top.clamp(min=1e-300) / 464)) + 1
        return torch.where(top > 0, x.clamp(min=-127), 0.0)

    low, high = exponents((z.abs() - d - 1e-30).clamp(min=0)), exponents(z.abs() + d + 1e-30)
    zero = torch.nn.functional.pad(z.abs(), (0, pad)).view(z.shape[0], -1, 32).amax(2) == 0
    assert (((X >= low) | (low == 0)) & (X <= high) | zero & (X == 0)).all()


def _product_case(pkg, M, N, K, lens, activation, options, bias, residual, device, pad=0):
    a, b, sa, sb, offs, gen = _inputs(M, N, K, lens, M + N)
    width = N // 2 if activation == "swiglu" else N
    bv = None if bias is None else torch.randn((len(lens), N), generator=gen).to(bias)
    res = torch.randn((M, width), generator=gen).to(torch.bfloat16) if residual else None
    args = (_strided(a, pad), _strided(b, pad), torch.tensor(sa).cuda(), torch.tensor(sb).cuda(), torch.tensor(offs).cuda(),
            None if bv is None else bv.cuda(), activation, None if res is None else _strided(res, pad))
    out, kept = pkg.grouped_gemm_fp8_bias_act(*args, keep_preact="mxfp8", zero_tail=True, **options)
    assert isinstance(kept, pkg.MXTensor) and kept.q.dtype == torch.float8_e4m3fn and tuple(kept.q.shape) == (M, N)
    z, _, size = orx.product(a.to(device), b.to(device), sa * sb, offs, None if bv is None else bv.to(device), activation, None, **options)
    _check_kept(pkg.MXTensor(kept.q.to(device), kept.scales.to(device)), z, size)
    plain = pkg.grouped_gemm_fp8_bias_act(*args, zero_tail=True, **options)
    both, pre = pkg.grouped_gemm_fp8_bias_act(*args, keep_preact=True, zero_tail=True, **options)
    # the same sums: what is kept is what the bf16 path rounds
    live = ~torch.isnan(z).any(1).cuda()
    back = pkg.dequantize_mx(kept)[live].double()
    power = torch.exp2(kept.scales[live].double() - 127).repeat_interleave(32, 1)[:, :N]
    got = pre[live].double()
    assert ((back - got).abs() <= (2.0 ** -4 + 2 * BF) * got.abs() + 2.0 ** -10 * power).all()
    for other in (plain, both):
        assert ((out.double() - other.double()).abs()[live] <= 0.02 * other.double().abs()[live] + 0.02).all()
    end = offs[-1]
    assert not out[end:].any() and not kept.q[end:].view(torch.uint8).any() and (kept.scales[end:] == 127).all()
    again = pkg.grouped_gemm_fp8_bias_act(*args, keep_preact="mxfp8", zero_tail=True, **options)
    assert torch.equal(out, again[0]) and torch.equal(kept.q.view(torch.uint8), again[1].q.view(torch.uint8))
    assert torch.equal(kept.scales, again[1].scales)


@pytest.mark.parametrize("M,N,K,lens", SHAPES)
@pytest.mark.parametrize("activation,options", ACTS)
@pytest.mark.parametrize("bias,residual", [(None, False), (torch.float32, True), (torch.bfloat16, False)])
def test_kept_values(pkg, M, N, K, lens, activation, options, bias, residual):
    _product_case(pkg, M, N, K, lens, activation, options, bias, residual, "cpu", 16 if residual else 0)


# tile rows with (swiglu, gelu and residual): of the shapes that reach every kernel
TILES = [(16, 16), (16, 16), (16, 16), (64, 64), (128, 128), (128, 128), (256, 128), (192, 192)]


@pytest.mark.parametrize("M,N,K,lens,rows", [(*case[:4], rows) for case, rows in zip(KERNELS, TILES)])
def test_every_kernel(pkg, M, N, K, lens, rows):
    from ggemm_asm_amd import _lib
    lib = _lib.load()
    for activation, options, residual, want in (("swiglu", GATE, False, rows[0]), ("gelu", {}, True, rows[1])):
        width = N // 2 if activation == "swiglu" else N
        assert lib.ggemm_mx_keep_tile_rows(len(lens), N, K, K, K, width, N, {"gelu": 2, "swiglu": 3}[activation], int(residual), M, 256) == want
        _product_case(pkg, M, N, K, lens, activation, options, torch.bfloat16, residual, "cuda")


@pytest.mark.parametrize("activation,options", ACTS)
def test_infinities_and_nan_stay_in_their_blocks(pkg, activation, options):
    for M, N, lens in ((12, 96, [5, 7]), (300, 352, [300]), (20000, 640, [20000])):
        a, b, sa, sb, offs, gen = _inputs(M, N, 64, lens, 5)
        a, b, offs = a.cuda(), b.cuda(), torch.tensor(offs).cuda()
        bias = torch.zeros((len(lens), N))
        bias[0, 40], bias[0, 70] = math.inf, math.nan
        _, kept = pkg.grouped_gemm_fp8_bias_act(a, b, torch.tensor(sa).cuda(), torch.tensor(sb).cuda(), offs, bias.cuda(), activation,
                                                keep_preact="mxfp8", **options)
        rows = torch.arange(M, device="cuda") < lens[0]
        want = torch.zeros_like(kept.scales, dtype=torch.bool)
        want[rows, 1], want[rows, 2] = True, True
        assert torch.equal(kept.scales == 255, want)


# --------------------------------------------------------------------------- the gradient

def _random_kept(pkg, M, N, seed, by_block=True):
    gen = torch.Generator().manual_seed(seed)
    z = torch.randn((M, N), generator=gen) * 3
    kept = pkg.quantize_mx(z.cuda(), "e4m3")
    if by_block:
        wide = torch.empty((kept.scales.shape[1], M + 5), dtype=torch.uint8, device="cuda")
        wide[:, :M] = kept.scales.t()
        kept = pkg.MXTensor(kept.q, wide.t()[:M])
    return kept, gen


def sum_of(v, offs):
    """The sums of v's rows, group by group."""
    return torch.stack([v[a:b].sum(0) for a, b in zip(offs, offs[1:])])


GRADS = [(1, 16, [1]), (70, 48, [0, 33, 1, 0, 30]), (300, 400, [65, 0, 128, 100]), (5003, 1424, [1200, 0, 1, 3700, 99]), (9, 5760, [4, 5])]


@pytest.mark.parametrize("M,N,lens", GRADS)
@pytest.mark.parametrize("activation,options", ACTS)
@pytest.mark.parametrize("by_block", [True, False])
def test_gradient(pkg, M, N, lens, activation, options, by_block):
    kept, gen = _random_kept(pkg, M, N, M + N, by_block)
    offs = [0]
    for n in lens:
        offs.append(offs[-1] + n)
    dout = torch.randn((M, N // 2 if activation == "swiglu" else N), generator=gen).to(torch.bfloat16).cuda()
    dev_offs = torch.tensor(offs).cuda()
    dpre, dbias = pkg.bias_act_backward(dout, kept, dev_offs, activation, **options)
    restored = pkg.dequantize_mx(kept)
    assert torch.equal(restored.double(), omx.decode(kept.q, kept.scales))
    same, same_bias = pkg.bias_act_backward(dout, restored, dev_offs, activation, **options)
    assert torch.equal(dpre, same)
    terms = (dpre.double().abs() * (1 + BF)).cumsum(0)
    terms = torch.cat((torch.zeros_like(terms[:1]), terms))
    total = terms[dev_offs[1:]] - terms[dev_offs[:-1]] + 1e-12 * terms[-1]
    n = (dev_offs[1:] - dev_offs[:-1])[:, None]
    assert ((dbias.double() - same_bias.double()).abs() <= (2 * n + 1) * 2.0 ** -24 * total).all()
    ref, ref_bias, size = orx.backward(dout.cpu(), restored.cpu(), offs, activation, **options)
    z = restored.cpu().double().abs() + 1
    factor = (z + options.get("shift", 0.0)).repeat_interleave(1, 1)
    if activation == "swiglu":
        pair = torch.maximum(z[:, 0::2], z[:, 1::2]) + options.get("shift", 0.0)
        factor = (pair * pair).repeat_interleave(2, 1) * options.get("slope", 1.0)
    d = dout.cpu().double().abs()
    d = d.repeat_interleave(2, 1) if activation == "swiglu" else d
    assert ((dpre.cpu().double() - ref).abs() <= 1.01 * BF * ref.abs() + 32 * 2.0 ** -23 * d * factor + 1e-30).all()
    assert ((dbias.cpu().double() - ref_bias).abs() <= ((2 * n + 1) * 2.0 ** -24 * total).cpu() + 32 * 2.0 ** -23 * sum_of(d * factor, offs)).all()
    assert not dpre[offs[-1]:].any()
    assert torch.equal(pkg.bias_act_backward(dout, kept, dev_offs, activation, bias_grad=False, **options)[0], dpre)


@pytest.mark.parametrize("G", [254, 255, 256, 2047])
@pytest.mark.parametrize("kept", [True, False])
def test_gradient_of_many_groups(pkg, G, kept):
    """Around the number of groups that a thread's one offset is enough for; ones of no rows, decreasing and negative offsets."""
    gen = torch.Generator().manual_seed(G)
    M, N = 700, 48
    z = pkg.quantize_mx(torch.randn((M, N), generator=gen).cuda(), "e4m3")
    restored = pkg.dequantize_mx(z)
    dout = torch.randn((M, N), generator=gen).to(torch.bfloat16).cuda()
    offs = torch.randint(0, M + 1, (G + 1,), generator=gen).sort()[0]
    for spoil in (False, True):
        if spoil:
            offs[G // 3], offs[G // 2], offs[-1] = -5, 0, M - 3
        dpre, dbias = pkg.bias_act_backward(dout, z if kept else restored, offs.cuda(), "silu")
        seen = offs.clamp(0, M).cummax(0)[0].tolist()
        ref, ref_bias, _ = orx.backward(dout.cpu(), restored.cpu(), seen, "silu")
        factor = restored.cpu().double().abs() + 1
        terms = dout.cpu().double().abs() * factor
        assert ((dpre.cpu().double() - ref).abs() <= 1.01 * BF * ref.abs() + 32 * 2.0 ** -23 * terms + 1e-30).all()
        count = torch.tensor([b - a for a, b in zip(seen, seen[1:])], dtype=torch.float64)[:, None]
        assert ((dbias.cpu().double() - ref_bias).abs() <= (32 + count) * 2.0 ** -23 * sum_of(terms, seen)).all()


def test_gradient_of_views_and_nan_blocks(pkg):
    kept, gen = _random_kept(pkg, 90, 96, 3)
    wide = torch.full((90, 120), 0xFF, dtype=torch.uint8, device="cuda")
    wide[:, 8:104] = kept.q.view(torch.uint8)
    odd = torch.full((90, 99), 0xFF, dtype=torch.uint8, device="cuda")
    odd[:, 3:] = kept.q.view(torch.uint8)
    dout = torch.randn((90, 96), generator=gen).to(torch.bfloat16).cuda()
    offs = torch.tensor([0, 50, 80]).cuda()
    want = pkg.bias_act_backward(dout, kept, offs, "silu")
    for raw in (wide[:, 8:104], odd[:, 3:]):
        got = pkg.bias_act_backward(dout, pkg.MXTensor(raw.view(torch.float8_e4m3fn), kept.scales), offs, "silu")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    scales = kept.scales.clone()
    scales[7, 1] = scales[85, 0] = 255
    dpre, dbias = pkg.bias_act_backward(dout, pkg.MXTensor(kept.q, scales), offs, "silu")
    nan = torch.zeros((90, 96), dtype=torch.bool, device="cuda")
    nan[7, 32:64] = True                                       # row 85 is of no group
    assert torch.equal(torch.isnan(dpre), nan)
    assert torch.equal(torch.isnan(dbias), torch.stack((nan[7], nan[8])))


def test_empty(pkg):
    kept = pkg.quantize_mx(torch.zeros((0, 64), device="cuda"), "e4m3")
    dpre, dbias = pkg.bias_act_backward(torch.zeros((0, 64), dtype=torch.bfloat16, device="cuda"), kept, torch.tensor([0, 0, 0]).cuda(), "silu")
    assert dpre.shape == (0, 64) and not dbias.any()
    a, b, sa, sb, offs, _ = _inputs(0, 64, 64, [0, 0], 1)
    out, kept = pkg.grouped_gemm_fp8_bias_act(a.cuda(), b.cuda(), torch.tensor(sa).cuda(), torch.tensor(sb).cuda(), torch.tensor(offs).cuda(),
                                              None, "silu", keep_preact="mxfp8")
    assert out.shape == (0, 64) and kept.q.shape == (0, 64) and kept.scales.shape == (0, 2)


# --------------------------------------------------------------------------- the layers

def _layer_inputs(seed, M=300, N=320, K=256, G=3):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((M, K), generator=gen).to(torch.bfloat16).cuda()
    w = (torch.randn((G, N, K), generator=gen) / 16).to(torch.bfloat16).cuda()
    bias = torch.randn((G, N), generator=gen).cuda()
    return x, w, bias, torch.tensor([0, 120, 120, 290]).cuda(), gen


@pytest.mark.parametrize("activation,options", ACTS)
def test_linear_layer_is_its_parts(pkg, activation, options):
    from ggemm_asm_amd.vark import weight_grad_fp8
    x, w, bias, offs, gen = _layer_inputs(1)
    dout = torch.randn((300, 160 if activation == "swiglu" else 320), generator=gen).to(torch.bfloat16).cuda()
    leaves = [t.clone().requires_grad_() for t in (x, w, bias)]
    out = pkg.grouped_linear_fp8(leaves[0], leaves[1], offs, bias=leaves[2], activation=activation, checkpoint="mxfp8", **options)
    out.backward(dout)
    plain = pkg.grouped_linear_fp8(x, w, offs, bias=bias, activation=activation, **options)
    assert torch.equal(out, plain)
    qx, sx, _ = pkg.quantize_fp8_tensorwise(x, row_align=128)
    qw, qwt, sw, _ = pkg.quantize_fp8_tensorwise_transpose(w, row_align=128)
    _, kept = pkg.grouped_gemm_fp8_bias_act(qx, qw, sx, sw, offs, bias, activation, keep_preact="mxfp8", zero_tail=True, **options)
    dy, db = pkg.bias_act_backward(dout, pkg.dequantize_mx(kept), offs, activation, **options)
    qdy, sdy, _ = pkg.quantize_fp8_tensorwise(dy, "e5m2", row_align=128)
    assert torch.allclose(leaves[2].grad, db, rtol=0, atol=float((2 * 290 + 1) * 2.0 ** -24 * (1 + BF) * dy.double().abs().sum(0).max()))
    assert torch.equal(leaves[0].grad, pkg.grouped_gemm_fp8_tensorwise(qdy, qwt, sdy, sw, offs, zero_tail=True))
    assert torch.equal(leaves[1].grad, weight_grad_fp8(qdy, qx, sdy, sx, offs))


def test_product_by_bias_and_residual(pkg):
    """The product's own gradients with the checkpoint that it returns."""
    a, b, sa, sb, offs, gen = _inputs(60, 64, 96, [20, 40], 4)
    bias = torch.randn((2, 64), generator=gen).cuda().requires_grad_()
    res = torch.randn((60, 64), generator=gen).to(torch.bfloat16).cuda().requires_grad_()
    args = (a.cuda(), b.cuda(), torch.tensor(sa).cuda(), torch.tensor(sb).cuda(), torch.tensor(offs).cuda())
    out, kept = pkg.grouped_gemm_fp8_bias_act(*args, bias, "gelu", res, keep_preact="mxfp8")
    assert isinstance(kept, pkg.MXTensor) and not kept.q.requires_grad
    dout = torch.randn((60, 64), generator=gen).to(torch.bfloat16).cuda()
    out.backward(dout)
    _, db = pkg.bias_act_backward(dout, kept, args[4], "gelu")
    assert torch.equal(bias.grad, db) and torch.equal(res.grad, dout)


def test_moe_layer(pkg):
    gen = torch.Generator().manual_seed(6)
    T, E, H, I = 200, 4, 128, 160
    x = torch.randn((T, H), generator=gen).to(torch.bfloat16).cuda()
    logits = torch.randn((T, E), generator=gen).cuda()
    w_up = (torch.randn((E, 2 * I, H), generator=gen) / 11).to(torch.bfloat16).cuda()
    w_down = (torch.randn((E, H, I), generator=gen) / 12).to(torch.bfloat16).cuda()
    dout = torch.randn((T, H), generator=gen).to(torch.bfloat16).cuda()
    got = []
    for checkpoint in (None, "mxfp8"):
        leaves = [t.clone().requires_grad_() for t in (x, logits, w_up, w_down)]
        out = pkg.moe_layer_fp8(*leaves, 2, checkpoint=checkpoint, **GATE)
        out.backward(dout)
        got.append((out, [t.grad for t in leaves]))
    assert torch.equal(got[0][0], got[1][0])
    # the down product's side does not read the checkpoint; the up product's gradients are taken at z off by 2^-4 of it at most
    assert torch.equal(got[0][1][1], got[1][1][1]) and torch.equal(got[0][1][3], got[1][1][3])
    for n in (0, 2):
        a, b = got[0][1][n].double(), got[1][1][n].double()
        assert not torch.equal(a, b) and (a - b).norm() <= 2.0 ** -3 * a.norm()


def test_captured(pkg):
    a, b, sa, sb, offs, gen = _inputs(300, 320, 256, [100, 0, 190], 8)
    args = (a.cuda(), b.cuda(), torch.tensor(sa).cuda(), torch.tensor(sb).cuda(), torch.tensor(offs).cuda())
    bias = torch.randn((3, 320), generator=gen).cuda()
    dout = torch.randn((300, 160), generator=gen).to(torch.bfloat16).cuda()

    def step():
        out, kept = pkg.grouped_gemm_fp8_bias_act(*args, bias, "swiglu", keep_preact="mxfp8", zero_tail=True, **GATE)
        return (out, kept.q.view(torch.uint8), kept.scales, *pkg.bias_act_backward(dout, kept, args[4], "swiglu", **GATE))

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = step()
    torch.cuda.synchronize()
    for k in range(3):
        bias.add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(c, e) for c, e in zip(captured, step()))


# units of 16, 32 and 64 rows: a thread goes through its eight rows in flight more than once, the last time with fewer
LONG = [(12000, 16, [3001, 0, 1, 8990, 5]), (25000, 32, [7, 24950, 13]), (50000, 64, [20003, 1, 29989])]


@pytest.mark.parametrize("M,rows,lens", LONG)
@pytest.mark.parametrize("activation,options", [("silu", {}), ("swiglu", GATE)])
def test_gradient_of_long_units(pkg, M, rows, lens, activation, options):
    """dpre the bits of the bf16 path. The sums against 64 bits: a term is off by 32 ulps of its factors, a sum of n terms by
    n 2^-24 of their magnitudes."""
    N, G = 5760, len(lens)
    assert pkg.load_library().ggemm_mx_act_workspace(M, G, N) == (M // rows + G) * N
    gen = torch.Generator(device="cuda").manual_seed(M)
    kept = pkg.quantize_mx(torch.randn((M, N), generator=gen, device="cuda") * 3, "e4m3")
    wide = torch.empty((kept.scales.shape[1], M), dtype=torch.uint8, device="cuda")
    kept = pkg.MXTensor(kept.q, wide.copy_(kept.scales.t()).t())
    width = N // 2 if activation == "swiglu" else N
    dout = torch.randn((M, width), generator=gen, device="cuda").to(torch.bfloat16)
    offs = [0]
    for n in lens:
        offs.append(offs[-1] + n)
    dev_offs = torch.tensor(offs).cuda()
    dpre, dbias = pkg.bias_act_backward(dout, kept, dev_offs, activation, **options)
    restored = pkg.dequantize_mx(kept)
    assert torch.equal(dpre, pkg.bias_act_backward(dout, restored, dev_offs, activation, **options)[0])
    assert not dpre[offs[-1]:].any()
    for g, (lo, hi) in enumerate(zip(offs, offs[1:])):
        z, d = restored[lo:hi].double(), dout[lo:hi].double()
        d = d.repeat_interleave(2, 1) if activation == "swiglu" else d
        terms = d * orx.act_grad(z, activation, **options)
        assert ((dpre[lo:hi].double() - terms).abs() <= 1.01 * BF * terms.abs() + 32 * 2.0 ** -23 * d.abs() * _factor(z, activation, options) + 1e-30).all()
        n = hi - lo
        err = (2.0 ** -24 * n * terms.abs() + 32 * 2.0 ** -23 * d.abs() * _factor(z, activation, options)).sum(0)
        assert ((dbias[g].double() - terms.sum(0)).abs() <= err).all()


def _factor(z, activation, options):
    """How large the factors are that a term is made of."""
    z = z.abs() + 1
    if activation != "swiglu":
        return z
    pair = torch.maximum(z[:, 0::2], z[:, 1::2]) + options.get("shift", 0.0)
    return (pair * pair).repeat_interleave(2, 1) * options.get("slope", 1.0)


# q and the gradient's rows past 2^32 bytes, by the tiles of 128, 192 and 256 rows; the last group's rows against the oracle
@pytest.mark.parametrize("N,K,activation,options,residual,rows",
                         [(5120, 128, "swiglu", GATE, False, 128), (5136, 1088, "gelu", {}, True, 192), (5120, 1088, "swiglu", GATE, False, 256)])
def test_kept_rows_past_32_bits(pkg, N, K, activation, options, residual, rows):
    M, last = 900000, 300
    width = N // 2 if activation == "swiglu" else N
    code = {"gelu": 2, "swiglu": 3}[activation]
    assert pkg.load_library().ggemm_mx_keep_tile_rows(2, N, K, K, K, width, N, code, int(residual), M, 256) == rows
    a, b, sa, sb, _, gen = _inputs(last, N, K, [0, last], 3)
    full = torch.zeros((M, K), dtype=torch.uint8, device="cuda")
    full[-last:] = a.view(torch.uint8).cuda()
    bias = torch.randn((2, N), generator=gen)
    tail = torch.randn((last, width), generator=gen).to(torch.bfloat16)
    res = None
    if residual:
        res = torch.zeros((M, width), dtype=torch.bfloat16, device="cuda")
        res[-last:] = tail.cuda()
    offs = torch.tensor([0, M - last, M]).cuda()
    out, kept = pkg.grouped_gemm_fp8_bias_act(full.view(a.dtype), b.cuda(), torch.tensor(sa).cuda(), torch.tensor(sb).cuda(), offs,
                                              bias.cuda(), activation, res, keep_preact="mxfp8", **options)
    del full, res
    z, ref, size = orx.product(a, b, sa * sb, [0, 0, last], bias, activation, tail if residual else None, **options)
    part = pkg.MXTensor(kept.q[-last:], kept.scales[-last:])
    _check_kept(pkg.MXTensor(part.q.cpu(), part.scales.cpu()), z, size)
    _check(out[-last:].cpu().double(), None, z, ref, size, activation, options, tail.double().abs() if residual else torch.zeros_like(ref))
    # every row before has the bias of its group alone: the same bytes all over
    assert (kept.q[:-last].view(torch.uint8) == kept.q[0].view(torch.uint8)).all() and (kept.scales[:-last] == kept.scales[0]).all()
    dout = torch.zeros_like(out)
    dout[-last:] = torch.randn((last, width), generator=gen).to(torch.bfloat16).cuda()
    dpre, dbias = pkg.bias_act_backward(dout, kept, offs, activation, **options)
    few, few_bias = pkg.bias_act_backward(dout[-last:], part, torch.tensor([0, 0, last]).cuda(), activation, **options)
    assert torch.equal(dpre[-last:], few) and not dpre[:-last].any() and not dbias[0].any()
    # the same terms in units of other lengths: each sum off by n 2^-24 of their magnitudes, known from their rounding to bf16
    assert ((dbias[1].double() - few_bias[1].double()).abs() <= 2 * last * 2.0 ** -24 * (1 + BF) * few.double().abs().sum(0)).all()
