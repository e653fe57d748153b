"""CPU checks of microscaled rows: the C ABI's refusals (before any HIP call), the torch ops' refusals, the choice of a
kernel, and the oracle against other ways to say the same."""
import math
import os
import re
import subprocess

import pytest
import torch

from conftest import ROOT
from oracle import mx_oracle as omx

FAKE = 0x100000


def test_header_symbols_exported(pkg):
    text = open(os.path.join(ROOT, "include", "ggemm_mx.h")).read()
    names = sorted(set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(ggemm_mx_\w+)\s*\(", text, re.M)))
    from ggemm_asm_amd import _lib
    assert names == sorted(_lib.MX_EXPORTS)
    lib = pkg.load_library()
    assert all(hasattr(lib, n) for n in names)


def _quantize(lib, **kw):
    a = dict(x=FAKE, dt=0, rows=10, cols=64, stride=64, fmt=0, q=FAKE, qs=64, s=FAKE, ss=2)
    a.update(kw)
    return lib.ggemm_mx_quantize(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(x=0), -1), (dict(q=0), -1), (dict(s=0), -1), (dict(dt=2), -8), (dict(fmt=2), -8), (dict(fmt=-1), -8),
    (dict(rows=-1), -2), (dict(cols=0), -2), (dict(cols=24), -2), (dict(stride=56), -3), (dict(stride=68), -3),
    (dict(dt=1, stride=66), -3), (dict(qs=56), -3), (dict(qs=68), -3), (dict(fmt=1, qs=28), -3), (dict(fmt=1, qs=34), -3),
    (dict(ss=1), -3), (dict(x=FAKE + 8), -4), (dict(q=FAKE + 4), -4), (dict(fmt=1, q=FAKE + 2), -4),
])
def test_quantize_validation(pkg, kw, rc):
    assert _quantize(pkg.load_library(), **kw) == rc


def _dequantize(lib, **kw):
    a = dict(q=FAKE, fmt=0, rows=10, cols=64, qs=64, s=FAKE, sr=2, sb=1, x=FAKE, dt=0, stride=64)
    a.update(kw)
    return lib.ggemm_mx_dequantize(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(x=0), -1), (dict(q=0), -1), (dict(s=0), -1), (dict(dt=3), -8), (dict(fmt=2), -8), (dict(rows=-1), -2),
    (dict(cols=40), -2), (dict(stride=60), -3), (dict(qs=63), -3), (dict(sr=-1), -3), (dict(sb=-1), -3), (dict(x=FAKE + 4), -4),
    (dict(q=FAKE + 1), -4),
])
def test_dequantize_validation(pkg, kw, rc):
    assert _dequantize(pkg.load_library(), **kw) == rc


def _product(lib, **kw):
    a = dict(a=FAKE, fmt=0, asc=FAKE, b=FAKE, bsc=FAKE, out=FAKE, bias=FAKE, bdt=0, res=FAKE, offs=FAKE, G=4, N=64, K=64, sa=64,
             sas=16, sbg=2048, sbn=32, sbsg=1024, sbsn=16, so=64, sr=64, act=0, slope=1.0, limit=7.0, shift=0.0, M=100, tail=0,
             tile=0)
    a.update(kw)
    return lib.ggemm_mx_product(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(a=0), -1), (dict(asc=0), -1), (dict(b=0), -1), (dict(bsc=0), -1), (dict(out=0), -1), (dict(offs=0), -1),
    (dict(fmt=2), -8), (dict(bdt=2), -8), (dict(act=4), -8), (dict(act=-1), -8), (dict(act=3, limit=0.0), -2),
    (dict(act=3, limit=math.nan), -2), (dict(G=0), -2), (dict(G=2048), -2), (dict(N=0), -2), (dict(N=40), -2),
    (dict(K=16), -2), (dict(K=80), -2), (dict(M=-1), -2), (dict(M=2 ** 31), -2), (dict(sa=48), -3), (dict(sa=72), -3),
    (dict(fmt=1, sa=16), -3), (dict(sas=0), -3), (dict(sas=24), -3), (dict(K=544, sa=544, sbn=272, sbg=17408), -3),
    (dict(sbn=16), -3), (dict(sbn=40), -3), (dict(sbsn=8), -3), (dict(sbg=2032), -3), (dict(sbsg=1008), -3), (dict(sbg=2056), -3),
    (dict(sa=2 ** 24), -2), (dict(sbsn=2 ** 24, sbsg=2 ** 30), -2), (dict(so=56), -3), (dict(so=68), -3), (dict(sr=56), -3),
    (dict(act=3, so=24), -3), (dict(a=FAKE + 8), -4), (dict(asc=FAKE + 8), -4), (dict(b=FAKE + 8), -4), (dict(bsc=FAKE + 4), -4),
    (dict(out=FAKE + 8), -4), (dict(bias=FAKE + 8), -4), (dict(res=FAKE + 8), -4), (dict(tile=48), -2), (dict(tile=-1), -2),
])
def test_product_validation(pkg, kw, rc):
    assert _product(pkg.load_library(), **kw) == rc


@pytest.mark.parametrize("kw,ok", [(dict(sbsn=32, sbsg=63 * 32 + 16), True), (dict(sbsn=32, sbsg=63 * 32), False),
                                   (dict(sbn=48, sbg=63 * 48 + 32), True), (dict(sbn=48, sbg=63 * 48 + 16), False)])
def test_product_takes_groups_that_follow_the_last_row_at_once(pkg, kw, ok):
    """A group's last row of scales need not be as far from the next group as rows from each other, as for values."""
    rc = _product(pkg.load_library(), **kw, M=0)
    assert (rc != -3) is ok


def _keep(lib, **kw):
    a = dict(a=FAKE, b=FAKE, out=FAKE, q=FAKE, s=FAKE, sa=FAKE, sb=FAKE, bias=FAKE, bdt=0, res=FAKE, offs=FAKE, G=4, N=64, K=32,
             sam=32, sbg=2048, sbn=32, so=64, sq=64, blk=100, sr=64, act=1, slope=1.0, limit=7.0, shift=0.0, M=100, tail=0)
    a.update(kw)
    return lib.ggemm_mx_keep_product(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(a=0), -1), (dict(q=0), -1), (dict(s=0), -1), (dict(out=0), -1), (dict(offs=0), -1), (dict(act=0), -8), (dict(act=4), -8),
    (dict(act=3, limit=0.0), -2), (dict(G=0), -2), (dict(N=40), -2), (dict(K=24), -2), (dict(M=-1), -2), (dict(sam=16), -3),
    (dict(so=56), -3), (dict(sq=48), -3), (dict(sq=72), -3), (dict(blk=99), -3), (dict(blk=2 ** 31), -2),
    (dict(sq=2 ** 24), -2), (dict(q=FAKE + 8), -4), (dict(out=FAKE + 8), -4), (dict(res=FAKE + 8), -4),
])
def test_keep_validation(pkg, kw, rc):
    assert _keep(pkg.load_library(), **kw) == rc


def test_kept_gradient_workspace(pkg):
    """A row of sums to every unit: units of 8 to 64 rows, a group's last one shorter."""
    f = pkg.load_library().ggemm_mx_act_workspace
    for M, G, N, rows in ((1, 1, 16, 8), (5003, 7, 1424, 8), (131072, 32, 5760, 64), (40000, 2047, 2048, 16)):
        assert f(M, G, N) == (M // rows + min(G, M)) * N
    assert f(0, 3, 64) == 64 and f(-1, 3, 64) == f(5, 0, 64) == f(5, 2048, 64) == 0


def _back(lib, **kw):
    a = dict(dout=FAKE, q=FAKE, s=FAKE, offs=FAKE, G=4, N=64, sd=64, sq=64, sr=2, sb=1, act=1, slope=1.0, limit=7.0, shift=0.0,
             M=100, dpre=FAKE, sdp=64, db=FAKE, ws=FAKE)
    a.update(kw)
    return lib.ggemm_mx_act_backward(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(dout=0), -1), (dict(q=0), -1), (dict(s=0), -1), (dict(dpre=0), -1), (dict(offs=0), -1), (dict(ws=0), -1),
    (dict(act=0), -8), (dict(act=9), -8), (dict(act=3, limit=0.0), -2), (dict(G=0), -2), (dict(N=24), -2), (dict(M=-1), -2),
    (dict(sd=56), -3), (dict(sq=56), -3), (dict(sq=68), -3), (dict(sdp=60), -3), (dict(sr=-1), -3), (dict(sb=-1), -3),
    (dict(dout=FAKE + 8), -4), (dict(q=FAKE + 4), -4), (dict(dpre=FAKE + 4), -4), (dict(db=FAKE + 8), -4), (dict(ws=FAKE + 8), -4),
])
def test_kept_gradient_validation(pkg, kw, rc):
    assert _back(pkg.load_library(), **kw) == rc


def test_choice_of_a_kernel(pkg):
    from ggemm_asm_amd import mx
    for fmt in ("e4m3", "e2m1"):
        assert [mx.tile_rows(fmt, 32, 5760, 2880, m) for m in (1, 256, 2048, 131072)] == [16, 32, 128, 256]
        assert all(mx.tile_rows(fmt, G, N, K, M) in mx.TILES[1:] for G in (1, 64, 2047) for N in (16, 5760) for K in (32, 8192)
                   for M in (1, 100, 10 ** 6))


WALK = """
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "mx_gemm.h"
int main(int argc, char** argv) {
  for (int i = 1; i + 1 < argc; i += 2) {
    const int cus = std::atoi(argv[i]), tiles = std::atoi(argv[i + 1]);
    const int run = ggemm::kXcds * ggemm::mid::kXcdRun, blocks = (tiles + run - 1) / run * run;
    const int grid = ggemm::mx::walk_grid(blocks, cus);
    std::vector<int> seen(tiles);
    for (int first = 0; first < grid; ++first)
      for (int b = first; b < blocks; b += grid) {
        const int t = ggemm::mid::tile_of_block(b);
        if (t >= tiles) break;
        ++seen[t];
      }
    int once = 0;
    for (int n : seen) once += n == 1;
    std::printf("%d\\n", grid >= 1 && once == tiles);
  }
}
"""


def test_walks_take_every_tile_on_any_number_of_cus(pkg, tmp_path):
    """The walk of the 256-row tiles in gemm_body: block, block + grid, .., up to the first that has no tile."""
    from ggemm_asm_amd import build
    if not os.path.exists(build.hipcc()):
        pytest.skip("hipcc not available")
    source, program = tmp_path / "walk.hip", tmp_path / "walk"
    source.write_text(WALK)
    subprocess.run([build.hipcc(), "-std=c++17", "--cuda-host-only", f"--offload-arch={build.ARCH}", "-I", build.CSRC, str(source),
                    "-o", str(program)], check=True, capture_output=True)
    cases = [(cus, tiles) for cus in (1, 7, 8, 32, 38, 64, 128, 228, 252, 256, 304) for tiles in (1, 255, 256, 257, 300, 700, 5000)]
    got = subprocess.run([str(program), *(str(v) for case in cases for v in case)], check=True, capture_output=True, text=True)
    assert [case for case, ok in zip(cases, got.stdout.split()) if ok != "1"] == [] and len(got.stdout.split()) == len(cases)


# --------------------------------------------------------------------------- the torch ops

def test_refusals(pkg):
    x = torch.zeros((4, 64))
    with pytest.raises(ValueError, match="fmt"):
        pkg.quantize_mx(x, "e5m2")
    with pytest.raises(TypeError):
        pkg.quantize_mx(x.double())
    with pytest.raises(ValueError, match="2 dimensions"):
        pkg.quantize_mx(x[0])
    with pytest.raises(ValueError, match="GPU"):
        pkg.quantize_mx(x)
    q, s = torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((4, 2), dtype=torch.uint8)
    with pytest.raises(TypeError):
        pkg.dequantize_mx(pkg.MXTensor(q, s), torch.float16)
    with pytest.raises(TypeError, match="e2m1"):
        pkg.dequantize_mx(pkg.MXTensor(q.float(), s))
    with pytest.raises(ValueError, match="scales"):
        pkg.dequantize_mx(pkg.MXTensor(q, s[:, :1]))
    with pytest.raises(ValueError, match="scales"):
        pkg.dequantize_mx(pkg.MXTensor(q, s.int()))
    with pytest.raises(ValueError, match="GPU"):
        pkg.dequantize_mx(pkg.MXTensor(q, s))
    b = pkg.MXTensor(q[None], s[None])
    offs = torch.tensor([0, 4])
    with pytest.raises(ValueError, match="2-D"):
        pkg.grouped_gemm_mx_bias_act(b, b, offs)
    with pytest.raises(TypeError, match="b must hold e2m1"):
        pkg.grouped_gemm_mx_bias_act(pkg.MXTensor(q, s), pkg.MXTensor(torch.zeros((1, 4, 64)).to(torch.float8_e4m3fn), s[None]), offs)
    with pytest.raises(ValueError, match="GPU"):
        pkg.grouped_gemm_mx_bias_act(pkg.MXTensor(q, s), b, offs)


@pytest.mark.parametrize("grad", [True, False])
def test_layer_refuses_an_unknown_checkpoint(pkg, grad):
    """Before anything else, on the path that keeps none too."""
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    w = torch.zeros((4, 64, 64), dtype=torch.bfloat16, requires_grad=grad)
    with pytest.raises(ValueError, match="checkpoint"):
        pkg.moe_layer_fp8(x, torch.zeros((2, 4)), w, w, 1, activation="silu", checkpoint="mxfp4")


@pytest.mark.parametrize("rows,features,first", [
    (131072, 512, False), (65536, 512, True), (16384, 512, True), (8192, 2880, True), (16384, 2880, False), (4096, 8192, True),
    (8192, 8192, False), (4, 8192, True),
])
def test_order_of_copying_and_quantizing_goes_by_bytes(pkg, rows, features, first):
    """The order that measured faster on either side of the crossing; 16384 rows of 512 values 20 us against 34, 8192 of 8192 values
    34 against 62, which a rule by rows alone gets wrong."""
    assert pkg.layer._copied_first(rows, features) is first


# --------------------------------------------------------------------------- the oracle

@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_exponents_are_the_smallest_that_fit(fmt):
    """Against the definition by trial: round with a table that goes on past the format's largest value."""
    v = omx.VALUES[fmt]
    longer = v + (v[-1] + (v[-1] - v[-2]), 2 * (v[-1] + (v[-1] - v[-2])))

    def fits(amax, x):
        s = math.ldexp(amax, -x)
        return s < longer[-1] and abs(s - v[-1]) < abs(s - longer[len(v)]) or s <= v[-1]

    gen = torch.Generator().manual_seed(1)
    some = torch.exp2(torch.rand(300, generator=gen, dtype=torch.float64) * 60 - 30).tolist()
    some += [m * 2.0 ** e for m in (1, 1.5, 1.75, 1.8125, 1.9999, 1.7499, 1.81249) for e in (-20, 0, 5, 100, 127)]
    for amax in some:
        amax = float(torch.tensor(amax, dtype=torch.float32))
        x = omx.exponent(amax, fmt)
        assert fits(amax, x) and not fits(amax, x - 1), (amax, x)
    assert omx.exponent(0.0, fmt) == 0 and omx.exponent(math.inf, fmt) == 128 and omx.exponent(math.nan, fmt) == 128
    assert omx.exponent(2.0 ** -149, fmt) == -127


def test_codes_match_torch_where_it_has_them():
    """e4m3 codes are those of torch's own cast of the scaled values; e2m1's are the nearest in its table."""
    gen = torch.Generator().manual_seed(2)
    x = torch.randn((50, 96), generator=gen) * torch.exp(3 * torch.randn((50, 1), generator=gen))
    codes, scales = omx.quantize(x, "e4m3")
    scaled = x.double() / torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    assert torch.equal(codes, scaled.float().to(torch.float8_e4m3fn).view(torch.uint8))
    codes, scales = omx.quantize(x, "e2m1")
    scaled = x.double() / torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    table = torch.tensor(omx.E2M1 + tuple(-v for v in omx.E2M1), dtype=torch.float64)
    got = table[codes.long()]
    assert ((got - scaled).abs() <= (scaled[..., None] - table).abs().amin(-1) + 1e-12).all()


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_storage_round_trip(fmt):
    gen = torch.Generator().manual_seed(3)
    q, s = omx.random_operand((6, 80), fmt, gen)
    v = omx.decode(q, s)
    assert v.shape == (6, 80)
    if fmt == "e2m1":                                     # the even column is the low half
        assert v[0, 0] == (omx.E2M1 + tuple(-x for x in omx.E2M1))[int(q[0, 0]) & 15] * 2.0 ** (int(s[0, 0]) - 127)
        assert v[5, 79] == (omx.E2M1 + tuple(-x for x in omx.E2M1))[int(q[5, 39]) >> 4] * 2.0 ** (int(s[5, 2]) - 127)
    else:
        assert v[3, 70] == float(q[3, 70]) * 2.0 ** (int(s[3, 2]) - 127)


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_quantization_error_is_half_a_step(fmt):
    """Nothing is off by more than the rounding of its own binade, the largest value of a block among it."""
    gen = torch.Generator().manual_seed(4)
    x = torch.randn((64, 256), generator=gen) * torch.exp(2 * torch.randn((64, 1), generator=gen))
    codes, scales = omx.quantize(x, fmt)
    back = omx.decode(omx.store(codes, fmt), scales)
    half, emin = (2.0 ** -2, 0) if fmt == "e2m1" else (2.0 ** -4, -6)
    power = torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    binade = torch.exp2(torch.floor(torch.log2(x.double().abs() / power)).clamp(min=emin)) * power
    assert ((back - x.double()).abs() <= half * binade * (1 + 1e-12)).all()


def test_product_by_loops():
    gen = torch.Generator().manual_seed(5)
    a, b = omx.random_operand((5, 64), "e4m3", gen, 120, 124), omx.random_operand((2, 16, 64), "e2m1", gen, 120, 124)
    a64, b64 = omx.decode(*a), omx.decode(*b)
    z, out, size = omx.product(a64, b64, "e4m3", [0, 2, 4], None, None, None)
    for r, g in ((0, 0), (1, 0), (2, 1), (3, 1)):
        for n in range(16):
            assert abs(float(z[r, n]) - sum(float(a64[r, k]) * float(b64[g, n, k]) for k in range(64))) < 1e-9 * float(size[r, n] + 1)
    assert torch.isnan(z[4]).all() and torch.equal(out[:4], z[:4])
