"""CPU checks of the product with an epilogue: the C ABI's refusals (before any HIP call), the torch ops' refusals, and
the oracle against differences."""
import math
import os
import re

import pytest
import torch

from conftest import ROOT
from oracle import product_oracle as orx

FAKE = 0x100000


def test_header_symbols_exported(pkg):
    text = open(os.path.join(ROOT, "include", "ggemm_product.h")).read()
    names = sorted(set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(ggemm_product_\w+)\s*\(", text, re.M)))
    from ggemm_asm_amd import _lib
    assert names == sorted(_lib.PRODUCT_EXPORTS)
    lib = pkg.load_library()
    assert all(hasattr(lib, n) for n in names)


def _product(lib, **kw):
    a = dict(a=FAKE, b=FAKE, out=FAKE, pre=FAKE, sa=FAKE, sb=FAKE, bias=FAKE, bdt=0, res=FAKE, offs=FAKE, G=4, N=64, K=32,
             sam=32, sbg=2048, sbn=32, so=64, sp=64, sr=64, act=0, slope=1.0, limit=7.0, shift=0.0, M=100, tail=0)
    a.update(kw)
    return lib.ggemm_product_fp8_bias_act(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(a=0), -1), (dict(b=0), -1), (dict(out=0), -1), (dict(sa=0), -1), (dict(sb=0), -1), (dict(offs=0), -1),
    (dict(bdt=2), -8), (dict(act=4), -8), (dict(act=-1), -8), (dict(act=3, limit=0.0), -2), (dict(act=3, limit=-1.0), -2),
    (dict(act=3, limit=math.nan), -2), (dict(G=0), -2), (dict(G=2048), -2), (dict(N=0), -2), (dict(N=40), -2),
    (dict(K=24), -2), (dict(M=-1), -2), (dict(M=2 ** 31), -2), (dict(sam=16), -3), (dict(sam=40), -3),
    (dict(sbn=16), -3), (dict(sbg=1024), -3), (dict(so=56), -3), (dict(so=68), -3), (dict(sp=56), -3),
    (dict(sr=56), -3), (dict(act=3, so=24), -3), (dict(act=3, sr=24), -3), (dict(a=FAKE + 8), -4), (dict(b=FAKE + 8), -4),
    (dict(out=FAKE + 8), -4), (dict(pre=FAKE + 8), -4), (dict(bias=FAKE + 8), -4), (dict(res=FAKE + 8), -4),
    (dict(sam=2 ** 24 * 16), -2),
])
def test_product_validation(pkg, kw, rc):
    assert _product(pkg.load_library(), **kw) == rc


def _back(lib, **kw):
    a = dict(dout=FAKE, pre=FAKE, offs=FAKE, G=4, N=64, sd=64, sp=64, act=1, slope=1.0, limit=7.0, shift=0.0, M=100,
             dpre=FAKE, sdp=64, db=FAKE, ws=FAKE)
    a.update(kw)
    return lib.ggemm_product_act_backward(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(dout=0), -1), (dict(pre=0), -1), (dict(dpre=0), -1), (dict(offs=0), -1), (dict(ws=0), -1), (dict(act=9), -8),
    (dict(act=3, limit=0.0), -2), (dict(G=0), -2), (dict(N=24), -2), (dict(M=-1), -2), (dict(sd=56), -3),
    (dict(sp=56), -3), (dict(sdp=60), -3), (dict(dout=FAKE + 8), -4), (dict(pre=FAKE + 2), -4), (dict(dpre=FAKE + 4), -4),
    (dict(db=FAKE + 8), -4), (dict(ws=FAKE + 8), -4),
])
def test_backward_validation(pkg, kw, rc):
    assert _back(pkg.load_library(), **kw) == rc


def test_workspace_holds_every_unit(pkg):
    """Units of a group are whole row blocks and one partial: M / rows and one more for each group that has rows."""
    f = pkg.load_library().ggemm_product_act_workspace
    assert f(-1, 4, 64) == 0 and f(10, 0, 64) == 0
    for M in (0, 1, 15, 16, 1000, 131072, 2 ** 31 - 256):
        for G in (1, 32, 2047):
            units = f(M, G, 64) // 64
            assert f(M, G, 64) % 64 == 0 and units >= max(1, min(G, M)) and units >= M // 256 // 4


@pytest.mark.parametrize("args,kw,rows", [
    ((32, 5760, 2880, 4, "swiglu"), {}, 16), ((8, 5760, 2880, 64, "gelu"), {}, 16), ((8, 5760, 2880, 128, "gelu"), {}, 64),
    ((32, 5760, 2880, 256, "swiglu"), {}, 64), ((64, 1536, 1024, 64), {}, 64), ((7, 2048, 1424, 5003, "gelu"), dict(residual=True), 128),
    ((32, 5760, 2880, 131072, "swiglu"), {}, 256), ((32, 5760, 2880, 131072, "swiglu"), dict(keep_preact=True), 256),
    ((32, 5760, 2880, 131072), {}, 256), ((32, 5760, 2880, 131072), dict(keep_preact=True), 192),
    ((32, 5760, 2880, 131072, "swiglu"), dict(residual=True), 192), ((32, 5760, 2880, 131072, "silu"), {}, 192),
    ((32, 5744, 2880, 131072, "swiglu"), {}, 192), ((300, 352, 96, 300), {}, 192)])
def test_kernel_choice(pkg, args, kw, rows):
    """The kernel by sizes, activation and what else the epilogue does; more than 256 groups only on the large tiles."""
    from ggemm_asm_amd import product
    assert product.tile_rows(*args, **kw) == rows


@pytest.fixture
def anywhere(pkg, monkeypatch):
    from ggemm_asm_amd import _lib, product
    monkeypatch.setattr(product, "_on_gpu", lambda *a: None)
    monkeypatch.setattr(_lib, "launch", lambda *a: pytest.fail("launched"))


E4, BF = torch.float8_e4m3fn, torch.bfloat16


@pytest.mark.parametrize("kw,exc", [
    (dict(a=torch.zeros((8, 32), dtype=torch.float8_e5m2)), TypeError), (dict(a=torch.zeros((8, 48), dtype=E4)), ValueError),
    (dict(a=torch.zeros((8, 64), dtype=E4)[:, ::2]), ValueError), (dict(a=torch.zeros(32, dtype=E4)), ValueError),
    (dict(b=torch.zeros((2, 64, 32), dtype=E4)), ValueError), (dict(sa=torch.ones(2)), ValueError),
    (dict(sb=torch.ones((), dtype=torch.float64)), ValueError), (dict(sb=torch.ones((), device="meta")), ValueError),
    (dict(offs=torch.zeros(4, dtype=torch.int32)), ValueError), (dict(offs=torch.zeros(4, dtype=torch.int64, device="meta")), ValueError),
    (dict(bias=torch.zeros(3, 63)), ValueError), (dict(bias=torch.zeros((3, 64), dtype=torch.float16)), ValueError),
    (dict(activation="relu"), ValueError), (dict(activation="silu", slope=2.0), ValueError),
    (dict(activation="gelu", limit=1.0), ValueError), (dict(shift=1.0), ValueError),
    (dict(activation="swiglu", limit=0.0), ValueError), (dict(activation="swiglu", limit=math.nan), ValueError),
    (dict(residual=torch.zeros((8, 32), dtype=BF)), ValueError), (dict(residual=torch.zeros(8, 64)), ValueError),
    (dict(activation="swiglu", residual=torch.zeros((8, 64), dtype=BF)), ValueError),
])
def test_product_refusals(pkg, anywhere, kw, exc):
    a = dict(a=torch.zeros((8, 32), dtype=E4), b=torch.zeros((3, 64, 32), dtype=E4), sa=torch.ones(()), sb=torch.ones(()),
             offs=torch.zeros(4, dtype=torch.int64))
    a.update(kw)
    with pytest.raises(exc):
        pkg.grouped_gemm_fp8_bias_act(*[a.pop(k) for k in ("a", "b", "sa", "sb", "offs")], **a)


@pytest.mark.parametrize("kw,exc", [
    (dict(dout=torch.zeros(8, 64)), TypeError), (dict(dout=torch.zeros((8, 40), dtype=BF)), ValueError),
    (dict(pre=None), ValueError), (dict(pre=torch.zeros((8, 32), dtype=BF)), ValueError), (dict(pre=torch.zeros(8, 64)), ValueError),
    (dict(activation="tanh"), ValueError), (dict(activation="swiglu"), ValueError), (dict(slope=2.0), ValueError),
    (dict(offs=torch.zeros(1, dtype=torch.int64)), ValueError),
])
def test_backward_refusals(pkg, anywhere, kw, exc):
    a = dict(dout=torch.zeros((8, 64), dtype=BF), pre=torch.zeros((8, 64), dtype=BF), offs=torch.zeros(4, dtype=torch.int64),
             activation="silu")
    a.update(kw)
    with pytest.raises(exc):
        pkg.bias_act_backward(a.pop("dout"), a.pop("pre"), a.pop("offs"), **a)


def test_ops_refuse_cpu_tensors(pkg):
    a, b = torch.zeros((8, 32), dtype=E4), torch.zeros((3, 64, 32), dtype=E4)
    offs = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU"):
        pkg.grouped_gemm_fp8_bias_act(a, b, torch.ones(()), torch.ones(()), offs)
    with pytest.raises(ValueError, match="GPU"):
        pkg.bias_act_backward(torch.zeros((8, 64), dtype=BF), None, offs)


@pytest.mark.parametrize("activation,options", [(None, {}), ("silu", {}), ("gelu", {}), ("swiglu", {}),
                                                ("swiglu", dict(slope=1.702, limit=2.0, shift=1.0))])
def test_oracle_gradient_against_differences(activation, options):
    z = torch.linspace(-4.01, 4.03, 64, dtype=torch.float64).view(4, 16)
    d = torch.linspace(-1, 1, 4 * (8 if activation == "swiglu" else 16), dtype=torch.float64).view(4, -1)
    dpre, _, _ = orx.backward(d, z, [0, 4], activation, **options)
    h = 1e-5
    for c in range(16):
        up, dn = z.clone(), z.clone()
        up[:, c] += h
        dn[:, c] -= h
        diff = ((orx.act(up, activation, **options) - orx.act(dn, activation, **options)) * d).sum(1) / (2 * h)
        torch.testing.assert_close(dpre[:, c], diff, atol=1e-8, rtol=0)


def test_few_rows_by_the_devices_cus(pkg):
    """The few-rows kernel is for launches whose mid tiles leave CUs without their two: on a quarter or an eighth of the
    CUs (a partitioned card) that is a quarter or an eighth of the tiles."""
    from ggemm_asm_amd import product
    for cus in (256, 128, 64, 32):
        for G in (1, 2, 4, 8, 16, 32):
            for N in (640, 1536, 2880, 5760):
                mid = G * -(-N // 128)
                rows = product.tile_rows(G, N, 4096, G, "silu", num_cus=cus)
                assert (rows == 16) == (mid <= 2 * cus), (cus, G, N, rows)
    # short rows of K: while the workgroups of 32 columns, three to a CU, leave half of the places free
    assert product.tile_rows(2, 1536, 1024, 2, num_cus=256) == 16 and product.tile_rows(2, 1536, 1024, 2, num_cus=32) == 64


def _unit_rows(M, N):
    """Rows of a unit as the launcher cuts them: 64, down to 16 while the units are fewer than 2048, more where they
    would be more than 2^22."""
    strips = -(-N // 8 // 256)
    rows = 64
    while rows > 16 and M // rows * strips < 2048:
        rows //= 2
    while M // rows * strips > 1 << 22:
        rows *= 2
    return rows


@pytest.mark.parametrize("N", [16, 64, 2064, 5760])
def test_workspace_of_the_worst_groups(pkg, N):
    """A group of n rows leaves ceil(n / rows) rows of partial sums. The most units that M rows of G groups can have, each
    group one row past a multiple of a unit, are within the workspace."""
    f = pkg.load_library().ggemm_product_act_workspace
    for M in (1, 2, 15, 16, 17, 1000, 4099, 32768, 131072, 131073, 10 ** 7, 2 ** 31 - 256):
        rows = _unit_rows(M, N)
        for G in (1, 2, 5, 32, 60, 2047):
            lens, left = [], M
            for _ in range(min(G, M)):                        # one row each: a unit each
                lens.append(1)
                left -= 1
            lens[0] += left // rows * rows                    # whole units
            left -= left // rows * rows
            if left:
                lens[-1] += left
            assert sum(lens) == M
            units, g = sum(-(-n // rows) for n in lens), min(G, M)
            assert units == g + (M - g) // rows               # the most: ceil(n / rows) is one more than (n - 1) // rows
            have = f(M, G, N)
            assert have % N == 0 and units * N <= have <= (M // rows + g) * N
