"""The grouped FP8 product with bias, activation and residual, and the gradient of bias and activation, on the GPU
against the 64-bit oracle.

Tolerances. z has the error of the matrix cores' fp8 sums (the oracle's bound, pinned by the products' own tests); an activation carries that error on by its slope, at most 1.2 times
the gate's reach, and adds a few ulps of exp2, reciprocal or erf (16 units of 2^-23 of the value and of z). The result
is rounded once to bf16: 2^-8. Gradients: the same ulps against the size of the factor, and in dbias the rounding
of a sum of `rows` terms, (rows / 64 + 16) 2^-24 of their magnitudes beside each term's 32 2^-23.
"""
import math

import pytest
import torch

from oracle import product_oracle as orx

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
BF = 2.0 ** -8
GATE = dict(slope=1.702, limit=7.0, shift=1.0)
ACTS = [(None, {}), ("silu", {}), ("gelu", {}), ("swiglu", {}), ("swiglu", GATE)]


def _inputs(M, N, K, lens, seed, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    a = (torch.randn((M, K), generator=gen) * 4).to(torch.float8_e4m3fn)
    b = (torch.randn((len(lens), N, K), generator=gen) * 4).to(torch.float8_e4m3fn)
    sa, sb = 0.25, 0.25 * std / math.sqrt(K)
    offs = [0]
    for n in lens:
        offs.append(offs[-1] + n)
    return a, b, sa, sb, offs, gen


def _strided(t, pad):
    """t on the GPU, its rows `pad` elements apart more than they are long."""
    wide = torch.zeros(tuple(t.shape[:-1]) + (t.shape[-1] + pad,), dtype=torch.uint8 if t.element_size() == 1 else t.dtype,
                       device="cuda")
    src = t.view(torch.uint8) if t.element_size() == 1 else t
    wide[..., :t.shape[-1]] = src.cuda()
    return (wide.view(t.dtype) if t.element_size() == 1 else wide)[..., :t.shape[-1]]


def _check(out, pre, z, ref, size, activation, options, extra):
    live = ~torch.isnan(z).any(1)
    dz = size[live]
    if pre is not None:
        assert ((pre[live] - z[live]).abs() <= dz + 1.01 * BF * z[live].abs() + 1e-30).all()
    if activation == "swiglu":
        zz = z[live].abs() + 1
        reach = torch.maximum(zz[:, 0::2], zz[:, 1::2]) + options.get("shift", 0.0)
        err = 1.2 * options.get("slope", 1.0) * (dz[:, 0::2] + dz[:, 1::2]) * reach + 16 * U * reach * reach
    else:
        err = 1.2 * dz + 16 * U * (z[live].abs() + 1) if activation else dz
    got, want = out[live], ref[live]
    bad = (got - want).abs() > err + 1.01 * BF * want.abs() + 4 * U * extra[live] + 1e-30
    assert not bad.any(), ((got - want).abs()[bad].max(), bad.nonzero()[:3])


# one row; groups empty, of one row and ragged; a tile and its edges; features below a tile, off its grid and over several
SHAPES = [(1, 16, 16, [0, 1, 0]), (4, 320, 2880, [1, 0, 1, 1, 0, 1]), (70, 48, 144, [0, 33, 1, 0, 36]),
          (300, 400, 272, [65, 0, 128, 100]), (257, 1040, 128, [257]), (64, 5760, 1424, [3] * 20),
          (5003, 336, 240, [1200, 0, 1, 3700, 99]), (4100, 2048, 160, [700] * 5 + [597])]


@pytest.mark.parametrize("M,N,K,lens", SHAPES)
@pytest.mark.parametrize("activation,options", ACTS)
@pytest.mark.parametrize("bias,residual,keep", [(None, False, True), (torch.float32, True, False), (torch.bfloat16, False, False),
                                                (torch.bfloat16, True, True)])
def test_product(pkg, M, N, K, lens, activation, options, bias, residual, keep):
    a, b, sa, sb, offs, gen = _inputs(M, N, K, lens, M + N)
    width = N // 2 if activation == "swiglu" else N
    bv = None if bias is None else torch.randn((len(lens), N), generator=gen).to(bias)
    res = torch.randn((M, width), generator=gen).to(torch.bfloat16) if residual else None
    pad = 16 if keep else 0
    dev = dict(device="cuda")
    args = (_strided(a, pad), _strided(b, pad), torch.tensor(sa, **dev), torch.tensor(sb, **dev), torch.tensor(offs, **dev),
            None if bv is None else bv.cuda(), activation, None if res is None else _strided(res, pad))
    got = pkg.grouped_gemm_fp8_bias_act(*args, keep_preact=keep, zero_tail=True, **options)
    out, pre = got if keep else (got, None)
    assert out.dtype == torch.bfloat16 and tuple(out.shape) == (M, width)
    z, ref, size = orx.product(a, b, sa * sb, offs, bv, activation, res, **options)
    _check(out.cpu().double(), None if pre is None else pre.cpu().double(), z, ref, size, activation, options,
           torch.zeros_like(ref) if res is None else res.double().abs())
    end = offs[-1]
    assert not out[end:].any() and (pre is None or not pre[end:].any())
    again = pkg.grouped_gemm_fp8_bias_act(*args, keep_preact=keep, zero_tail=True, **options)
    assert torch.equal(out, again[0] if keep else again)


def test_more_groups_than_the_small_tiles_take(pkg):
    """300 groups: the launch goes to the persistent kernel whatever its rows."""
    lens = [1, 0, 2] * 100
    a, b, sa, sb, offs, gen = _inputs(sum(lens), 352, 96, lens, 9)
    bias = torch.randn((300, 352), generator=gen)
    for activation, options in ACTS:
        out, pre = pkg.grouped_gemm_fp8_bias_act(a.cuda(), b.cuda(), torch.tensor(sa).cuda(), torch.tensor(sb).cuda(),
                                                 torch.tensor(offs).cuda(), bias.cuda(), activation, keep_preact=True, **options)
        z, ref, size = orx.product(a, b, sa * sb, offs, bias, activation, None, **options)
        _check(out.cpu().double(), pre.cpu().double(), z, ref, size, activation, options, torch.zeros_like(ref))


# rows, features, group lengths, tile rows with (bias, swiglu, swiglu and z, gelu and residual): every kernel with every
# epilogue it has, at a group's edge and past a row tile, K of a half step and of several batches
KERNELS = [(1, 320, 2880, [0, 1, 0], (16,) * 4), (30, 5760, 2064, [17, 0, 13], (16,) * 4), (40, 1040, 8208, [9, 11, 3, 16, 1], (16,) * 4),
           (150, 1040, 144, [80, 70], (64,) * 4), (2500, 3200, 192, [1000, 0, 1499], (128,) * 4),
           (20000, 2560, 320, [256, 19001, 0, 700], (256, 256, 128, 192)), (16000, 1280, 1088, [15999], (256, 256, 256, 128)),
           (20000, 2096, 2880, [5000, 4999, 0, 10001], (192,) * 4)]


@pytest.mark.parametrize("M,N,K,lens,rows", KERNELS)
def test_every_kernel(pkg, M, N, K, lens, rows):
    """On the GPU's own fp64 (these are larger than the CPU's oracle takes quickly): the same formulas and bounds."""
    from ggemm_asm_amd import product
    a, b, sa, sb, offs, gen = _inputs(M, N, K, lens, M + N)
    G = len(lens)
    bias = torch.randn((G, N), generator=gen).to(torch.bfloat16).cuda()
    cases = [(None, {}, False, False), ("swiglu", GATE, False, False), ("swiglu", GATE, True, False), ("gelu", {}, False, True)]
    res = torch.randn((M, N), generator=gen).to(torch.bfloat16).cuda()
    a, b, dev_offs = a.cuda(), b.cuda(), torch.tensor(offs).cuda()
    for (activation, options, keep, residual), want in zip(cases, rows):
        assert product.tile_rows(G, N, K, M, activation, keep_preact=keep, residual=residual) == want
        got = pkg.grouped_gemm_fp8_bias_act(a, b, torch.tensor(sa).cuda(), torch.tensor(sb).cuda(), dev_offs, bias, activation,
                                            res if residual else None, keep_preact=keep, zero_tail=True, **options)
        out, pre = got if keep else (got, None)
        z, ref, size = orx.product(a, b, sa * sb, offs, bias, activation, res if residual else None, **options)
        _check(out.double(), None if pre is None else pre.double(), z, ref, size, activation, options,
               res.double().abs() if residual else torch.zeros_like(ref))
        assert not out[offs[-1]:].any() and (pre is None or not pre[offs[-1]:].any())


@pytest.mark.parametrize("activation,options", ACTS)
def test_clamped_and_extreme_values(pkg, activation, options):
    """z far outside the activations' bends and the clamp: nothing overflows on the way."""
    a, b, sa, sb, offs, _ = _inputs(40, 64, 64, [40], 5, std=200.0)
    out, pre = pkg.grouped_gemm_fp8_bias_act(a.cuda(), b.cuda(), torch.tensor(sa).cuda(), torch.tensor(sb).cuda(),
                                             torch.tensor(offs).cuda(), None, activation, keep_preact=True, **options)
    z, ref, size = orx.product(a, b, sa * sb, offs, None, activation, None, **options)
    assert torch.isfinite(out).all() and z.abs().max() > 300
    _check(out.cpu().double(), pre.cpu().double(), z, ref, size, activation, options, torch.zeros_like(ref))


def test_nan_and_infinite_bias(pkg):
    """NaN stays NaN through the clamp, and only in its own columns."""
    a, b, sa, sb, offs, _ = _inputs(20, 64, 32, [20], 6)
    bias = torch.zeros((1, 64))
    bias[0, 10], bias[0, 21], bias[0, 40] = math.nan, math.nan, math.inf
    for activation, options in ACTS:
        out = pkg.grouped_gemm_fp8_bias_act(a.cuda(), b.cuda(), torch.tensor(sa).cuda(), torch.tensor(sb).cuda(),
                                            torch.tensor(offs).cuda(), bias.cuda(), activation, **options).cpu()
        _, ref, _ = orx.product(a, b, sa * sb, offs, bias, activation, None, **options)
        assert torch.equal(torch.isnan(out), torch.isnan(ref)), activation
        fin = torch.isfinite(ref)
        assert torch.equal(torch.isfinite(out), fin)


def test_empty_and_offsets_past_the_rows(pkg):
    a, b, sa, sb, offs, _ = _inputs(100, 64, 32, [30, 70], 8)
    one = torch.tensor(1.0).cuda()
    out = pkg.grouped_gemm_fp8_bias_act(a[:0].cuda(), b.cuda(), one, one, torch.tensor([0, 0, 0]).cuda(), None, "swiglu")
    assert tuple(out.shape) == (0, 32)
    cut = pkg.grouped_gemm_fp8_bias_act(a[:50].cuda(), b.cuda(), one, one, torch.tensor([0, 30, 10 ** 12]).cuda())
    full = pkg.grouped_gemm_fp8_bias_act(a.cuda(), b.cuda(), one, one, torch.tensor(offs).cuda())
    assert torch.equal(cut, full[:50])
    with pytest.raises(pkg.GGemmError):
        pkg.grouped_gemm_fp8_bias_act(a.cuda(), b.cuda(), one, one, torch.tensor([0, 50, 40]).cuda(), validate=True)


def test_strides_of_single_rows_and_groups(pkg):
    """Where there is one row or one group its stride is whatever the view has."""
    a, b, sa, sb, offs, _ = _inputs(3, 64, 96, [3], 12)
    one = torch.tensor(1.0).cuda()
    wide = torch.zeros((3, 104), dtype=torch.uint8, device="cuda")
    wide[:, :96] = a.view(torch.uint8).cuda()
    row = wide.view(a.dtype)[:1, :96]
    group = b.cuda().as_strided((1, 64, 96), (8, 96, 1))
    assert row.stride(0) % 16 and group.stride(0) == 8
    got = pkg.grouped_gemm_fp8_bias_act(row, group, one, one, torch.tensor([0, 1]).cuda())
    want = pkg.grouped_gemm_fp8_bias_act(a[:1].cuda(), b.cuda(), one, one, torch.tensor([0, 1]).cuda())
    assert torch.equal(got, want)


BACK = [(1, 16, [1]), (7, 48, [0, 3, 0, 2]), (100, 2064, [33, 1, 60]), (1000, 320, [0, 999]), (2500, 5760, [400, 0, 1, 2000, 50]),
        (40000, 64, [13000, 27000]), (600, 32, [2] * 300)]


@pytest.mark.parametrize("M,N,lens", BACK)
@pytest.mark.parametrize("activation,options", ACTS)
def test_gradient(pkg, M, N, lens, activation, options):
    gen = torch.Generator().manual_seed(M + N)
    width = N // 2 if activation == "swiglu" else N
    pre = (torch.randn((M, N), generator=gen) * 4).to(torch.bfloat16)
    dout = torch.randn((M, width), generator=gen).to(torch.bfloat16)
    offs = [0]
    for n in lens:
        offs.append(offs[-1] + n)
    dev_offs = torch.tensor(offs).cuda()
    dpre, dbias = pkg.bias_act_backward(_strided(dout, 8), _strided(pre, 8), dev_offs, activation, **options)
    ref, rbias, size = orx.backward(dout, pre, offs, activation, **options)
    # each factor's error against its largest term
    term = dout.double().abs()
    term = term.repeat_interleave(2, 1) if activation == "swiglu" else term
    other = pre.double().abs()
    if activation == "swiglu":
        other = torch.maximum(other[:, 0::2], other[:, 1::2]).repeat_interleave(2, 1)
    term = term * (other + 2) ** 2 if activation == "swiglu" else term * (other + 2)
    if activation is None:
        assert torch.equal(dpre.cpu(), dout)
    else:
        end = offs[-1]
        assert ((dpre.cpu().double() - ref).abs() <= 1.01 * BF * ref.abs() + 32 * U * term + 1e-30).all()
        assert not dpre[end:].any()
    for g, (lo, hi) in enumerate(zip(offs, offs[1:])):
        tol = 32 * U * term[lo:hi].sum(0) + ((hi - lo) / 64 + 16) * 2.0 ** -24 * size[g]
        assert ((dbias[g].cpu().double() - rbias[g]).abs() <= tol).all()
    same, none = pkg.bias_act_backward(dout.cuda(), pre.cuda(), dev_offs, activation, bias_grad=False, **options)
    assert none is None and torch.equal(same, dpre)
    assert torch.equal(pkg.bias_act_backward(dout.cuda(), pre.cuda(), dev_offs, activation, **options)[1], dbias)


def test_gradient_of_no_rows_and_odd_offsets(pkg):
    one = torch.ones((6, 16), dtype=torch.bfloat16, device="cuda")
    _, dbias = pkg.bias_act_backward(one[:0], one[:0], torch.tensor([0, 0, 0]).cuda(), "silu")
    assert tuple(dbias.shape) == (2, 16) and not dbias.any()
    # offsets that begin late, fall and leave the rows: rows belong to the first group that holds them
    offs = torch.tensor([1, 4, 2, 99]).cuda()
    dpre, dbias = pkg.bias_act_backward(one, None, offs)
    assert dbias[:, 0].tolist() == [3.0, 0.0, 2.0]
    zero = torch.zeros_like(one)
    dpre, _ = pkg.bias_act_backward(one, zero, offs, "silu")
    assert dpre[:, 0].tolist() == [0.0, 0.5, 0.5, 0.5, 0.5, 0.5]


# z, the result and the residual past 2^32 bytes; the last group's rows against the oracle
@pytest.mark.parametrize("K,activation,options,keep,residual,rows",
                         [(128, None, {}, False, False, 256), (128, "swiglu", GATE, True, False, 128),
                          (1088, "swiglu", GATE, True, False, 256), (128, "gelu", {}, False, True, 192)])
def test_rows_past_32_bits(pkg, K, activation, options, keep, residual, rows):
    from ggemm_asm_amd import product
    M, N, last = 900000, 2560, 300
    a, b, sa, sb, _, gen = _inputs(last, N, K, [0, last], 3)
    full = torch.zeros((M, K), dtype=torch.uint8, device="cuda")
    full[-last:] = a.view(torch.uint8).cuda()
    bias = torch.randn((2, N), generator=gen)
    tail = torch.randn((last, N), generator=gen).to(torch.bfloat16)
    res = None
    if residual:
        res = torch.zeros((M, N), dtype=torch.bfloat16, device="cuda")
        res[-last:] = tail.cuda()
    assert product.tile_rows(2, N, K, M, activation, keep_preact=keep, residual=residual) == rows
    got = pkg.grouped_gemm_fp8_bias_act(full.view(a.dtype), b.cuda(), torch.tensor(sa).cuda(), torch.tensor(sb).cuda(),
                                        torch.tensor([0, M - last, M]).cuda(), bias.cuda(), activation, res, keep_preact=keep, **options)
    out, pre = got if keep else (got, None)
    z, ref, size = orx.product(a, b, sa * sb, [0, 0, last], bias, activation, tail if residual else None, **options)
    _check(out[-last:].cpu().double(), None if pre is None else pre[-last:].cpu().double(), z, ref, size, activation, options,
           tail.double().abs() if residual else torch.zeros_like(ref))


# weights of 256 groups, 2^32 bytes and more
@pytest.mark.parametrize("M,N,K,rows", [(2, 4096, 4224, 16), (600, 4096, 4224, 64), (20000, 2560, 6720, 256)])
def test_weights_past_32_bits(pkg, M, N, K, rows):
    from ggemm_asm_amd import product
    G = 256
    a, b, sa, sb, _, gen = _inputs(M, N, K, [1], 4)
    weights = torch.zeros((G, N, K), dtype=torch.uint8, device="cuda")
    weights[-1] = b[0].view(torch.uint8).cuda()
    bias = torch.randn((1, N), generator=gen)
    biases = torch.zeros((G, N), device="cuda")
    biases[-1] = bias[0].cuda()
    offs = torch.zeros(G + 1, dtype=torch.int64)
    offs[-1] = M
    assert product.tile_rows(G, N, K, M, "swiglu") == rows
    out = pkg.grouped_gemm_fp8_bias_act(a.cuda(), weights.view(b.dtype), torch.tensor(sa).cuda(), torch.tensor(sb).cuda(), offs.cuda(),
                                        biases, "swiglu", **GATE)
    part = slice(max(0, M - 300), M)
    z, ref, size = orx.product(a[part], b, sa * sb, [0, part.stop - part.start], bias, "swiglu", None, **GATE)
    _check(out[part].cpu().double(), None, z, ref, size, "swiglu", GATE, torch.zeros_like(ref))


def test_gradient_past_32_bits(pkg):
    M, N, last = 900000, 2560, 300
    gen = torch.Generator().manual_seed(5)
    tail, dtail = torch.randn((last, N), generator=gen).to(torch.bfloat16), torch.randn((last, N), generator=gen).to(torch.bfloat16)
    pre, dout = torch.zeros((M, N), dtype=torch.bfloat16, device="cuda"), torch.zeros((M, N), dtype=torch.bfloat16, device="cuda")
    pre[-last:], dout[-last:] = tail.cuda(), dtail.cuda()
    dpre, dbias = pkg.bias_act_backward(dout, pre, torch.tensor([0, M - last, M]).cuda(), "gelu")
    # the same rows by themselves: equal in dpre; the sums' units are cut alike from the group's first row, but may be of fewer rows
    few, fewb = pkg.bias_act_backward(dtail.cuda(), tail.cuda(), torch.tensor([0, 0, last]).cuda(), "gelu")
    assert torch.equal(dpre[-last:], few) and not dpre[:-last].any() and not dbias[0].any()
    want = few.double().sum(0)
    err = few.double().abs().sum(0) * (BF / 2 + (last + 16) * U)      # few is rounded, the sums are not
    assert ((dbias[1].double() - want).abs() <= err).all() and ((fewb[1].double() - want).abs() <= err).all()


@pytest.mark.parametrize("M,N,K,lens,rows", [(30, 5760, 2064, [17, 0, 13], 16), (150, 1040, 144, [80, 70], 64),
                                             (2500, 3200, 192, [1000, 0, 1499], 128), (20000, 2096, 2880, [5000, 4999, 0, 10001], 192),
                                             (16000, 1280, 1088, [15999], 256)])
@pytest.mark.parametrize("options", [{}, GATE])
@pytest.mark.parametrize("keep", [False, True])
def test_special_values_on_every_kernel(pkg, M, N, K, lens, rows, options, keep):
    """Gates switched off by a bias near the lowest finite value give zeros, whatever the up half; NaN stays in its
    columns; infinities do what the formula says. Other columns are finite."""
    from ggemm_asm_amd import product
    a, b, sa, sb, offs, _ = _inputs(M, N, K, lens, M)
    G = len(lens)
    assert product.tile_rows(G, N, K, M, "swiglu", keep_preact=keep) == rows
    bias = torch.zeros((G, N))
    off = [0, 14, 322, N - 2]                             # gate columns, of several waves and tiles
    for c in off[:2]:
        bias[:, c] = -3.2e38
    for c in off[2:]:
        bias[:, c] = -5e37
    bias[:, 41] = math.nan                               # an up half
    bias[:, 100] = math.nan                              # a gate
    bias[:, 200] = -math.inf                             # -inf times a sigmoid of 0
    got = pkg.grouped_gemm_fp8_bias_act(a.cuda(), b.cuda(), torch.tensor(sa).cuda(), torch.tensor(sb).cuda(),
                                        torch.tensor(offs).cuda(), bias.cuda(), "swiglu", keep_preact=keep, **options)
    out = (got[0] if keep else got)[:offs[-1]].float()
    nan = torch.zeros(N // 2, dtype=torch.bool, device="cuda")
    nan[[20, 50, 100]] = True
    assert torch.equal(torch.isnan(out).all(0), nan) and torch.equal(torch.isnan(out).any(0), nan)
    assert not out[:, [c // 2 for c in off]].any()
    assert torch.isfinite(out[:, ~nan]).all()
    if keep:
        assert torch.equal(torch.isnan(got[1][:offs[-1]]).all(0).nonzero().flatten().cpu(), torch.tensor([41, 100]))
        assert (got[1][:offs[-1], off] < -4e37).all()


def test_bias_gradient_of_the_most_rows(pkg):
    """2^31 - 256 rows in one group (and a few before it): their number plus a unit's rows is past 31 bits."""
    M = 2 ** 31 - 256
    dout = torch.ones((M, 16), dtype=torch.bfloat16, device="cuda")
    _, dbias = pkg.bias_act_backward(dout, None, torch.tensor([0, M]).cuda())
    assert (dbias == float(M)).all()                      # every partial sum is a multiple of 256 below 2^24 of them
    _, dbias = pkg.bias_act_backward(dout, None, torch.tensor([0, 256, M]).cuda())
    assert (dbias[0] == 256).all() and (dbias[1] == float(M - 256)).all()


@pytest.mark.parametrize("activation,options", ACTS)
@pytest.mark.parametrize("bias_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("keep", [False, True])
def test_gradients_of_bias_and_residual(pkg, activation, options, bias_dtype, keep):
    """The result as without gradients, bit for bit; the bias' gradient that of the kept z, the residual's the result's own
    in the groups' rows and zero outside them. Tolerances as in test_gradient, and one rounding to the bias' type."""
    lens = [0, 33, 1, 0, 36]
    M, N, K = 77, 48, 144
    a, b, sa, sb, offs, gen = _inputs(M, N, K, lens, 21)
    width = N // 2 if activation == "swiglu" else N
    args = (a.cuda(), b.cuda(), torch.tensor(sa).cuda(), torch.tensor(sb).cuda(), torch.tensor(offs).cuda())
    bias = torch.randn((len(lens), N), generator=gen).to(bias_dtype).cuda()
    res = torch.randn((M, width), generator=gen).to(torch.bfloat16).cuda()
    dout = torch.randn((M, width), generator=gen).to(torch.bfloat16).cuda()
    plain, pre = pkg.grouped_gemm_fp8_bias_act(*args, bias, activation, res, keep_preact=True, zero_tail=True, **options)
    bias.requires_grad_()
    res.requires_grad_()
    got = pkg.grouped_gemm_fp8_bias_act(*args, bias, activation, res, keep_preact=keep, zero_tail=True, **options)
    out = got[0] if keep else got
    assert torch.equal(out, plain) and (not keep or torch.equal(got[1], pre))
    out.backward(dout)
    _, want, size = orx.backward(dout.cpu(), pre.cpu(), offs, activation, **options)
    half = BF if bias_dtype == torch.bfloat16 else 0.0
    reach = (float(pre[:offs[-1]].abs().max()) + 2) ** 2 * float(dout.abs().max()) * max(lens)
    assert bias.grad.dtype == bias_dtype
    assert ((bias.grad.cpu().double() - want).abs() <= 32 * U * reach + 17 * 2.0 ** -24 * size + 1.01 * half * want.abs()).all()
    assert torch.equal(res.grad[:offs[-1]], dout[:offs[-1]]) and not res.grad[offs[-1]:].any()


def test_gradient_of_gates_far_below_zero(pkg):
    """Where the gate is closed its gradient is zero, and where it nearly is their product is what counts, however large the
    up half times dout would be by themselves."""
    pre = torch.zeros((3, 16), dtype=torch.bfloat16)
    pre[0, 0::2], pre[0, 1::2] = -3e38, 1e10
    pre[1, 0::2], pre[1, 1::2] = -64.0, 1e20
    pre[2, 0::2], pre[2, 1::2] = -3e38, -1e37
    dout = torch.full((3, 8), 1e30, dtype=torch.bfloat16)
    offs = [0, 1, 2, 3]
    dpre, dbias = pkg.bias_act_backward(dout.cuda(), pre.cuda(), torch.tensor(offs).cuda(), "swiglu", shift=1.0)
    ref, rbias, _ = orx.backward(dout, pre, offs, "swiglu", shift=1.0)
    assert torch.isfinite(ref).all() and torch.isfinite(dpre).all() and torch.isfinite(dbias).all()
    # sigmoid(-64): the exponent's rounding, 64 log2 e 2^-24 ln 2 = 3.8e-6, and the difference 1 - 64 of two terms
    for got, want, half in ((dpre, ref, BF), (dbias, rbias, 0.0)):
        assert ((got.cpu().double() - want).abs() <= (1e-5 + half) * want.abs()).all()
