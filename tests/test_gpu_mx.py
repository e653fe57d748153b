"""Microscaled rows on the GPU against the 64-bit oracle.

Quantization is byte work: every code and scale has to be the oracle's; values come back exactly. Products: the bound of
``mx_oracle.product`` on z, carried through the activation and rounded once to bf16 (2^-8), as in the tests of the
product with per-tensor scales; where nothing but the product and its rounding is left, their 2-norm is off by the
rounding's 2^-8 and half as much for the sums.
"""
import math

import pytest
import torch

from oracle import mx_oracle as omx

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
BF = 2.0 ** -8
GATE = dict(slope=1.702, limit=7.0, shift=1.0)
ACTS = [(None, {}), ("silu", {}), ("gelu", {}), ("swiglu", {}), ("swiglu", GATE)]
FORMATS = ("e2m1", "e4m3")


def _rows(shape, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen) * torch.exp(2 * torch.randn(shape[-1], generator=gen))
    return x.to(dtype)


def _same(kept, x, fmt):
    codes, scales = omx.quantize(x.reshape(-1, x.shape[-1]), fmt)
    want = omx.store(codes, fmt).view(torch.uint8)
    got = kept.q.cpu().reshape(-1, kept.q.shape[-1]).view(torch.uint8)
    assert torch.equal(kept.scales.cpu().reshape(scales.shape), scales)
    assert torch.equal(got, want), (got != want).nonzero()[:4]


# --------------------------------------------------------------------------- rows to blocks and back

@pytest.mark.parametrize("shape", [(1, 16), (1, 32), (3, 48), (1, 2880), (7, 2880), (37, 1424), (2, 5, 96), (33, 4112)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize(pkg, shape, dtype, fmt):
    x = _rows(shape, dtype, sum(shape))
    kept = pkg.quantize_mx(x.cuda(), fmt)
    assert kept.q.shape[:-1] == x.shape[:-1] and kept.scales.shape == x.shape[:-1] + (-(-shape[-1] // 32),)
    _same(kept, x, fmt)
    aligned = pkg.quantize_mx(x.cuda(), fmt, row_align=128)
    assert torch.equal(aligned.q.view(torch.uint8), kept.q.view(torch.uint8)) and aligned.q.stride(-2) % 128 == 0
    assert torch.equal(aligned.scales, kept.scales)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt", FORMATS)
def test_special_values(pkg, dtype, fmt):
    """Blocks whose largest value lies on and beside every bend of the exponent's rule, ties of every code, zeros of both
    signs, subnormal numbers, the ends of the range, infinities and NaN."""
    up = 1.75 if fmt == "e2m1" else 1.8125
    step = 2.0 ** (-7 if dtype == torch.bfloat16 else -23)
    table = torch.tensor(omx.VALUES[fmt])
    rows = []
    for e in (-127, -126, -125, -30, 0, 9, 127):
        for m in (1.0, up - step, up, up + step, 2 - step):
            if e < -126:
                m = round(m / 2 * 128) / 128 * 2            # what subnormal bf16 holds
            rows.append([m * 2.0 ** e if e > -127 else m * 2.0 ** -127] + [(-1) ** i * m * 2.0 ** (e - i % 12) if e > -100 else 0.0
                                                                          for i in range(31)])
    for lo in range(0, len(table) - 1, 16):                  # ties, the largest value first to hold the exponent
        part = (table[lo:lo + 16][:-1] + table[lo:lo + 16][1:]) / 2
        rows.append([float(table[-1])] + part.tolist() + (-part).tolist() + [0.0] * (31 - 2 * len(part)))
    rows += [[0.0] * 32, [-0.0] * 32, [0.0] * 31 + [-2.0 ** -133], [math.inf] + [1.0] * 31, [1.0] * 31 + [-math.inf],
             [math.nan] + [3.0] * 31, [0.0] * 16 + [-math.nan] * 16]
    x = torch.tensor(rows, dtype=torch.float64).to(dtype)
    kept = pkg.quantize_mx(x.cuda(), fmt)
    _same(kept, x, fmt)
    for out in (torch.float32, torch.bfloat16):
        got = pkg.dequantize_mx(kept, out).cpu()
        want = omx.decode(kept.q.cpu(), kept.scales.cpu()).to(out)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_every_code_and_scale_comes_back(pkg, fmt, out):
    scales = torch.arange(256, dtype=torch.int16).to(torch.uint8)
    codes = torch.arange(16 if fmt == "e2m1" else 256, dtype=torch.int16).to(torch.uint8)
    q = codes.repeat(256, 2 if fmt == "e2m1" else 1)
    stored = omx.store(q, fmt)
    s = scales[:, None].repeat(1, q.shape[1] // 32)
    got = pkg.dequantize_mx(pkg.MXTensor(stored.cuda(), s.cuda()), out).cpu()
    want = omx.decode(stored, s).to(out)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


def test_rows_of_other_strides(pkg):
    """Rows that are views: of a wider buffer, not 16-byte aligned, expanded, transposed; scales by blocks first."""
    wide = _rows((9, 320), torch.bfloat16, 3).cuda()
    for x in (wide[:, :96], wide[:, 8:104], wide[:, 3:99], wide[:1, :96].expand(5, 96), wide[:, :32].t().contiguous().t(),
              wide[0:0, :96], wide[3:4, 16:48]):
        for fmt in FORMATS:
            kept = pkg.quantize_mx(x, fmt)
            _same(kept, x.cpu(), fmt)
            by_block = kept.scales.t().contiguous().t()
            assert torch.equal(pkg.dequantize_mx(pkg.MXTensor(kept.q, by_block)), pkg.dequantize_mx(kept))
            other = torch.empty((x.shape[0], kept.q.shape[1] + 3), dtype=torch.uint8, device="cuda")[:, 3:]
            other.copy_(kept.q.view(torch.uint8))
            moved = pkg.MXTensor(other.view(kept.q.dtype), kept.scales)
            assert torch.equal(pkg.dequantize_mx(moved), pkg.dequantize_mx(kept))


def test_nothing_outside_is_written(pkg):
    """q and scales as views of buffers whose other bytes stay what they were, through the C ABI."""
    from ggemm_asm_amd import _lib
    x = _rows((5, 48), torch.bfloat16, 4).cuda()
    for code, width in ((0, 48), (1, 24)):
        q = torch.full((7, 64), 0xA5, dtype=torch.uint8, device="cuda")
        s = torch.full((7, 16), 0x5A, dtype=torch.uint8, device="cuda")
        _lib.launch("ggemm_mx_quantize", x.device, 48, x.data_ptr(), 0, 5, 48, 48, code, q[1:].data_ptr(), 64, s[1:].data_ptr(), 16)
        assert (q[0] == 0xA5).all() and (q[6] == 0xA5).all() and (q[1:6, width:] == 0xA5).all()
        assert (s[0] == 0x5A).all() and (s[6] == 0x5A).all() and (s[1:6, 2:] == 0x5A).all() and not (s[1:6, :2] == 0x5A).all()


# --------------------------------------------------------------------------- the product

def _offs(lens):
    offs = [0]
    for n in lens:
        offs.append(offs[-1] + n)
    return offs


def _laid_out(t, pad, fill=0xFF):
    """t on the GPU in rows of 16-byte multiples, `pad` more, filled up with `fill`: NaN codes and scales."""
    raw = t.view(torch.uint8)
    wide = torch.full(tuple(raw.shape[:-1]) + (-(-raw.shape[-1] // 16) * 16 + pad,), fill, dtype=torch.uint8, device="cuda")
    wide[..., :raw.shape[-1]] = raw.cuda()
    return wide.view(t.dtype)[..., :raw.shape[-1]]


def _check(out, z, ref, size, activation, options, extra):
    live = ~torch.isnan(z).any(1)
    dz = size[live]
    if activation == "swiglu":
        zz = z[live].abs() + 1
        reach = torch.maximum(zz[:, 0::2], zz[:, 1::2]) + options.get("shift", 0.0)
        err = 1.2 * options.get("slope", 1.0) * (dz[:, 0::2] + dz[:, 1::2]) * reach + 16 * U * reach * reach
    else:
        err = 1.2 * dz + 16 * U * (z[live].abs() + 1) if activation else dz
    got, want = out[live], ref[live]
    bad = ~((got - want).abs() <= err + 1.01 * BF * want.abs() + 4 * U * extra[live] + 1e-30)
    assert not bad.any(), ((got - want).abs()[bad].max(), bad.sum(), bad.nonzero()[:3])
    if activation is None:
        assert (got - want).norm() <= 1.5 * BF * want.norm() + 1e-30


def _case(M, N, K, lens, fmt, seed):
    gen = torch.Generator().manual_seed(seed)
    a = omx.random_operand((M, K), fmt, gen)
    if fmt == "e4m3":                                    # codes as quantized activations have them: 2^-7 .. 448
        a = (torch.randn((M, K), generator=gen).mul(60).to(torch.float8_e4m3fn), a[1])
    b = omx.random_operand((len(lens), N, K), "e2m1", gen, 112, 122)
    return a, b, _offs(lens), gen


# one row; groups empty, of one row and ragged; a tile and its edges; features below a tile, off its grid and over several;
# one block of K, half a stage, odd stages
SHAPES = [(1, 16, 32, [0, 1, 0]), (4, 320, 2880, [1, 0, 1, 1, 0, 1]), (70, 48, 160, [0, 33, 1, 0, 36]),
          (300, 400, 288, [65, 0, 128, 100]), (257, 1040, 128, [257]), (64, 576, 1440, [3] * 20),
          (700, 336, 544, [300, 0, 1, 257, 99])]


@pytest.mark.parametrize("M,N,K,lens", SHAPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tile", [0, 16, 32, 64, 128, 256])
def test_product(pkg, M, N, K, lens, fmt, tile):
    a, b, offs, gen = _case(M, N, K, lens, fmt, M + N)
    pad = 16 if tile else 0
    da, db = (pkg.MXTensor(_laid_out(q, pad), _laid_out(s, pad)) for q, s in (a, b))
    a64, b64 = omx.decode(*a), omx.decode(*b)
    for k, (activation, options) in enumerate(ACTS):
        width = N // 2 if activation == "swiglu" else N
        bias = (None, torch.randn((len(lens), N), generator=gen), torch.randn((len(lens), N), generator=gen).bfloat16())[k % 3]
        res = torch.randn((M, width), generator=gen).bfloat16() if k % 2 else None
        args = (da, db, torch.tensor(offs).cuda(), None if bias is None else bias.cuda(), activation,
                None if res is None else res.cuda())
        out = pkg.grouped_gemm_mx_bias_act(*args, zero_tail=True, tile=tile, **options)
        assert out.dtype == torch.bfloat16 and tuple(out.shape) == (M, width)
        z, ref, size = omx.product(a64, b64, fmt, offs, bias, activation, res, **options)
        _check(out.cpu().double(), z, ref, size, activation, options, torch.zeros_like(ref) if res is None else res.double().abs())
        assert not out[offs[-1]:].any()
        assert torch.equal(out, pkg.grouped_gemm_mx_bias_act(*args, zero_tail=True, tile=tile, **options))


# more rows than a tile, K of many stages, several bands and rounds: on the GPU's own fp64
LARGE = [(5000, 2048, 1440, [1200, 0, 1, 3700, 99]), (20000, 2880, 2880, [256, 19001, 0, 700]), (9000, 5760, 2880, [300] * 30),
         (3000, 1040, 5760, [1000, 1999])]


@pytest.mark.parametrize("M,N,K,lens", LARGE)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tile", [0, 32, 64, 128, 256])
def test_large_product(pkg, M, N, K, lens, fmt, tile):
    a, b, offs, gen = _case(M, N, K, lens, fmt, M + N)
    da, db = (pkg.MXTensor(_laid_out(q, 0), _laid_out(s, 0)) for q, s in (a, b))
    a64, b64 = omx.decode(*da), omx.decode(*db)
    bias = torch.randn((len(lens), N), generator=gen).bfloat16().cuda()
    for activation, options in ((None, {}), ("swiglu", GATE)):
        out = pkg.grouped_gemm_mx_bias_act(da, db, torch.tensor(offs).cuda(), bias, activation, zero_tail=True, tile=tile, **options)
        z, ref, size = omx.product(a64, b64, fmt, offs, bias, activation, None, **options)
        _check(out.double(), z, ref, size, activation, options, torch.zeros_like(ref))
        assert not out[offs[-1]:].any()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tile", [16, 32, 64, 128, 256])
def test_many_groups_and_odd_offsets(pkg, fmt, tile):
    """More groups than lanes, and the most there may be; offsets that start late, fall, leave the tensor or are negative."""
    lens = [1, 0, 2, 5] * 75
    a, b, offs, _ = _case(sum(lens) + 3, 48, 96, lens, fmt, 5)
    a64, b64 = omx.decode(*a), omx.decode(*b)
    da, db = (pkg.MXTensor(_laid_out(q, 0), _laid_out(s, 0)) for q, s in (a, b))
    out = pkg.grouped_gemm_mx_bias_act(da, db, torch.tensor(offs).cuda(), zero_tail=True, tile=tile)
    z, ref, size = omx.product(a64, b64, fmt, offs, None, None, None)
    _check(out.cpu().double(), z, ref, size, None, {}, torch.zeros_like(ref))
    assert not out[offs[-1]:].any()

    gen = torch.Generator().manual_seed(8)
    many = torch.sort(torch.randint(0, 900, (2048,), generator=gen)).values.tolist()
    for offs in ([40, 60, 30, 90, 1000, 20], [-5, 30, 20, 50, 50, 10 ** 12], [0, 0, 0, 0, 0, 0], many):
        G, M = len(offs) - 1, 800 if len(offs) > 100 else 120
        a, b = omx.random_operand((M, 64), fmt, gen, 120, 124), omx.random_operand((G, 32, 64), "e2m1", gen, 112, 122)
        da, db = (pkg.MXTensor(_laid_out(q, 0), _laid_out(s, 0)) for q, s in (a, b))
        base = torch.full((M, 32), 7.0, dtype=torch.bfloat16, device="cuda")
        top, seen = [], 0
        for o in offs:
            seen = max(seen, min(max(o, 0), M))
            top.append(seen)
        out = pkg.grouped_gemm_mx_bias_act(da, db, torch.tensor(offs).cuda(), residual=base, tile=tile)
        z, ref, size = omx.product(omx.decode(*a), omx.decode(*b), fmt, top, None, None, base.cpu())
        _check(out.cpu().double(), z, ref, size, None, {}, torch.full_like(ref, 7.0))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tile", [16, 32, 64, 128, 256])
def test_nan_blocks_reach_their_rows_alone(pkg, fmt, tile):
    a, b, offs, _ = _case(90, 64, 352, [50, 40], fmt, 6)
    a[1][7, 3] = 255
    b[1][1, 20, 10] = 255
    da, db = (pkg.MXTensor(_laid_out(q, 0), _laid_out(s, 0)) for q, s in (a, b))
    out = pkg.grouped_gemm_mx_bias_act(da, db, torch.tensor(offs).cuda(), tile=tile).cpu()
    want = torch.zeros((90, 64), dtype=torch.bool)
    want[7] = True
    want[50:, 20] = True
    assert torch.equal(torch.isnan(out), want)


def test_any_layout(pkg):
    """Operands that the kernels cannot read where they are give the same results as laid out ones."""
    a, b, offs, gen = _case(40, 48, 1440, [30, 10], "e4m3", 7)
    dev_offs = torch.tensor(offs).cuda()
    want = pkg.grouped_gemm_mx_bias_act(pkg.MXTensor(_laid_out(a[0], 0), _laid_out(a[1], 0)),
                                        pkg.MXTensor(_laid_out(b[0], 0), _laid_out(b[1], 0)), dev_offs)
    plain = pkg.MXTensor(a[0].cuda(), a[1].cuda()), pkg.MXTensor(b[0].cuda(), b[1].cuda())
    assert torch.equal(want, pkg.grouped_gemm_mx_bias_act(*plain, dev_offs))

    def odd(t):
        wide = torch.full(tuple(t.shape[:-1]) + (t.shape[-1] + 7,), 255, dtype=torch.uint8, device="cuda")
        wide[..., 5:-2] = t.view(torch.uint8).cuda()
        return wide[..., 5:-2].view(t.dtype)

    assert torch.equal(want, pkg.grouped_gemm_mx_bias_act(pkg.MXTensor(odd(a[0]), odd(a[1])), pkg.MXTensor(odd(b[0]), odd(b[1])), dev_offs))
    # groups last in memory, and one weight for all experts
    last = [t.permute(1, 2, 0).contiguous().permute(2, 0, 1) for t in plain[1]]
    assert torch.equal(want, pkg.grouped_gemm_mx_bias_act(plain[0], pkg.MXTensor(*last), dev_offs))
    one = pkg.MXTensor(plain[1].q[:1].expand(2, -1, -1), plain[1].scales[:1].expand(2, -1, -1))
    copy = pkg.MXTensor(one.q.contiguous(), one.scales.contiguous())
    assert torch.equal(pkg.grouped_gemm_mx_bias_act(plain[0], one, dev_offs), pkg.grouped_gemm_mx_bias_act(plain[0], copy, dev_offs))


def test_quantized_rows_through_the_product(pkg):
    """quantize_mx's own layout, activations and weights, as a layer uses them."""
    gen = torch.Generator().manual_seed(11)
    x = torch.randn((77, 2880), generator=gen).bfloat16()
    w = (torch.randn((3, 320, 2880), generator=gen) / 50).bfloat16()
    offs = [0, 30, 30, 77]
    kb = pkg.quantize_mx(w.cuda(), "e2m1", row_align=128)
    for fmt in FORMATS:
        ka = pkg.quantize_mx(x.cuda(), fmt, row_align=128)
        out = pkg.grouped_gemm_mx_bias_act(ka, kb, torch.tensor(offs).cuda())
        z, ref, size = omx.product(omx.decode(*ka), omx.decode(*kb), fmt, offs, None, None, None)
        _check(out.double(), z, ref, size, None, {}, torch.zeros_like(ref))


def test_captured_and_on_another_stream(pkg):
    a, b, offs, gen = _case(300, 640, 2880, [100, 0, 200], "e4m3", 12)
    x = _rows((300, 2880), torch.bfloat16, 13).cuda()
    db = pkg.MXTensor(_laid_out(b[0], 0), _laid_out(b[1], 0))
    dev_offs = torch.tensor(offs).cuda()

    def step():
        kept = pkg.quantize_mx(x, "e4m3", row_align=128)
        return pkg.dequantize_mx(kept), pkg.grouped_gemm_mx_bias_act(kept, db, dev_offs, activation="swiglu", zero_tail=True, **GATE)

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = step()
    torch.cuda.synchronize()
    for k in range(3):
        x.copy_(_rows((300, 2880), torch.bfloat16, 13 + k).cuda())
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(c, e) for c, e in zip(captured, eager))
        if k == 0:
            assert all(torch.equal(c, e) for c, e in zip(on_side, eager))


def test_past_32_bit_offsets(pkg):
    """Rows and weights beyond 2^32 bytes: quantized, restored and multiplied at both ends."""
    rows, cols = 420000, 5760
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
    some = [0, 1, rows // 2, rows - 2, rows - 1]
    x[some] = _rows((len(some), cols), torch.bfloat16, 14).cuda()
    for fmt in FORMATS:
        kept = pkg.quantize_mx(x, fmt)
        _same(pkg.MXTensor(kept.q[some], kept.scales[some]), x[some].cpu(), fmt)
        assert int((kept.scales != 127).any(1).sum()) == len(some)
        assert torch.equal(pkg.dequantize_mx(kept)[some].double(), omx.decode(kept.q[some], kept.scales[some]))
    del x, kept
    G, N, K = 600, 5760, 2880
    q = torch.zeros((G, N, 1536), dtype=torch.uint8, device="cuda")[..., :K // 2]
    s = torch.full((G, N, 96), 127, dtype=torch.uint8, device="cuda")[..., :K // 32]
    gen = torch.Generator().manual_seed(15)
    for g in (0, 599):
        bq, bs = omx.random_operand((N, K), "e2m1", gen, 112, 122)
        q[g], s[g] = bq.cuda(), bs.cuda()
    a = omx.random_operand((40, K), "e2m1", gen)
    offs = [0, 20] + [20] * 598 + [40]
    for tile in (16, 256):
        out = pkg.grouped_gemm_mx_bias_act(pkg.MXTensor(a[0].cuda(), a[1].cuda()), pkg.MXTensor(q, s), torch.tensor(offs).cuda(), tile=tile)
        a64 = omx.decode(*a).cuda()
        for g, lo in ((0, 0), (599, 20)):
            z, ref, size = omx.product(a64[lo:lo + 20], omx.decode(q[g:g + 1], s[g:g + 1]), "e2m1", [0, 20], None, None, None)
            _check(out[lo:lo + 20].double(), z, ref, size, None, {}, torch.zeros_like(ref))


# more tiles of 256 rows than CUs, so that workgroups walk over them: K of two and of three stages of either format, the last one
# whole, half full or of one block
@pytest.mark.parametrize("K", [160, 256, 288, 384, 512, 544, 768])
@pytest.mark.parametrize("fmt", FORMATS)
def test_walks_of_few_stages(pkg, fmt, K):
    M, N, lens = 20000, 2896, [256, 19001, 0, 700]
    a, b, offs, gen = _case(M, N, K, lens, fmt, K)
    da, db = (pkg.MXTensor(_laid_out(q, 0), _laid_out(s, 0)) for q, s in (a, b))
    bias = torch.randn((len(lens), N), generator=gen).cuda()
    out = pkg.grouped_gemm_mx_bias_act(da, db, torch.tensor(offs).cuda(), bias, zero_tail=True, tile=256)
    z, ref, size = omx.product(omx.decode(*da), omx.decode(*db), fmt, offs, bias, None, None)
    _check(out.double(), z, ref, size, None, {}, torch.zeros_like(ref))
    assert not out[offs[-1]:].any()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("activation,options,dtype,residual", [("gelu", {}, torch.float32, True), ("silu", {}, None, True),
                                                               ("swiglu", GATE, torch.float32, True), (None, {}, torch.float32, False)])
def test_walks_with_every_operand(pkg, fmt, activation, options, dtype, residual):
    """A later tile's bias comes into the place of the last one's (for e2m1 of its results too) and its residual is read while the
    next stages are in flight."""
    M, N, K, lens = LARGE[1]
    a, b, offs, gen = _case(M, N, K, lens, fmt, 21)
    da, db = (pkg.MXTensor(_laid_out(q, 0), _laid_out(s, 0)) for q, s in (a, b))
    bias = None if dtype is None else torch.randn((len(lens), N), generator=gen).to(dtype).cuda()
    res = torch.randn((M, N // 2 if activation == "swiglu" else N), generator=gen).bfloat16().cuda() if residual else None
    out = pkg.grouped_gemm_mx_bias_act(da, db, torch.tensor(offs).cuda(), bias, activation, res, zero_tail=True, tile=256, **options)
    z, ref, size = omx.product(omx.decode(*da), omx.decode(*db), fmt, offs, bias, activation, res, **options)
    _check(out.double(), z, ref, size, activation, options, torch.zeros_like(ref) if res is None else res.double().abs())
    assert not out[offs[-1]:].any()


def test_rows_past_32_bit_offsets(pkg):
    """Rows of a (e4m3), of the residual and of the result past 2^32 bytes, by every tile."""
    M, N, K, last = 900000, 2560, 4800, 300
    a, b, _, gen = _case(last, N, K, [0, last], "e4m3", 16)
    q = torch.zeros((M, K), dtype=torch.uint8, device="cuda")
    s = torch.full((M, 160), 127, dtype=torch.uint8, device="cuda")[:, :K // 32]
    q[-last:], s[-last:] = a[0].view(torch.uint8).cuda(), a[1].cuda()
    tail = torch.randn((last, N), generator=gen).bfloat16()
    res = torch.zeros((M, N), dtype=torch.bfloat16, device="cuda")
    res[-last:] = tail.cuda()
    bias = torch.randn((2, N), generator=gen)
    db = pkg.MXTensor(_laid_out(b[0], 0), _laid_out(b[1], 0))
    z, ref, size = omx.product(omx.decode(*a), omx.decode(*b), "e4m3", [0, 0, last], bias, None, tail)
    for tile in (16, 32, 64, 128, 256):
        out = pkg.grouped_gemm_mx_bias_act(pkg.MXTensor(q.view(torch.float8_e4m3fn), s), db, torch.tensor([0, M - last, M]).cuda(), bias.cuda(),
                                           None, res, tile=tile)
        _check(out[-last:].cpu().double(), z, ref, size, None, {}, tail.double().abs())
        assert (out[:-last] == bias[0].bfloat16().cuda()).all()


@pytest.mark.parametrize("tile", [16, 32, 64, 128, 256])
def test_groups_that_follow_the_last_row_at_once(pkg, tile):
    """Scales of a group whose rows are 64 bytes apart, the next group 16 bytes after the last one: read where they are."""
    a, b, offs, _ = _case(40, 48, 480, [25, 15], "e4m3", 22)
    da, db = (pkg.MXTensor(_laid_out(q, 0), _laid_out(s, 0)) for q, s in (a, b))
    pitch, group = 64, 47 * 64 + 16
    buffer = torch.full((2 * group,), 255, dtype=torch.uint8, device="cuda")
    tight = buffer.as_strided((2, 48, 15), (group, pitch, 1))
    tight.copy_(db.scales)
    dev_offs = torch.tensor(offs).cuda()
    want = pkg.grouped_gemm_mx_bias_act(da, db, dev_offs, tile=tile)
    assert torch.equal(want, pkg.grouped_gemm_mx_bias_act(da, pkg.MXTensor(db.q, tight), dev_offs, tile=tile))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tile", [16, 32, 64, 128, 256])
def test_scales_at_the_ends_of_their_range(pkg, fmt, tile):
    """Every power that a scale can hold on one side, and on the other one that brings the product back; zeros under the largest
    scales stay zeros, and products below fp32 vanish."""
    M, N, K = 32, 32, 64
    for s in (0, 1, 2, 40, 127, 200, 253, 254):
        for d in (-3, 0, 4):
            t = 254 - s + d
            if not 0 <= t <= 254:
                continue
            a, b, offs, gen = _case(M, N, K, [M], fmt, 300 + s)
            a[1].fill_(s), b[1].fill_(t)
            out = pkg.grouped_gemm_mx_bias_act(pkg.MXTensor(_laid_out(a[0], 0), _laid_out(a[1], 0)),
                                               pkg.MXTensor(_laid_out(b[0], 0), _laid_out(b[1], 0)), torch.tensor(offs).cuda(), tile=tile)
            z, ref, size = omx.product(omx.decode(*a), omx.decode(*b), fmt, offs, None, None, None)
            _check(out.cpu().double(), z, ref, size, None, {}, torch.zeros_like(ref))
    zero = torch.zeros_like(a[0].view(torch.uint8)).view(a[0].dtype)
    for q, s in ((zero, 254), (a[0], 0)):
        a[1].fill_(s), b[1].fill_(s)
        out = pkg.grouped_gemm_mx_bias_act(pkg.MXTensor(_laid_out(q, 0), _laid_out(a[1], 0)),
                                           pkg.MXTensor(_laid_out(b[0], 0), _laid_out(b[1], 0)), torch.tensor(offs).cuda(), tile=tile)
        assert not out.any()
