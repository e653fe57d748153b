"""CPU checks of the wide tiles that keep z in 8 bits (KEEP8_CONFIGS of ggemm-asm_amd/csrc/gen_vark_wide.py), before any GPU
launch: their per-tile assembly runs lane by lane as in test_product_wide_host, with the instructions that it has more.
Every kept byte and scale has to be the oracle's for the fp32 z of the same program.
"""
import numpy as np
import pytest
import torch

import test_product_wide_host as P
import test_vark_wide_host as W
from oracle import mx_oracle as omx

GEN, M32, _f, _bits = W.GEN, W.M32, P._f, P._bits
CFG = GEN.KEEP8_CONFIGS[0]
PRE8, SCALES = 0x7A0000000000, 0x790000000000


def _e4m3(x):
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy().astype(np.uint32)


def _program():
    """The program, its new instructions in a form that the emulation's one-result operations take."""
    prog, labels = P._program(CFG)
    out = []
    for op, a in prog:
        if op == "v_cvt_scalef32_pk_fp8_f32":
            hi = "op_sel" in a[3]
            a = [a[0], a[1], a[2], a[3].split()[0]] + ([a[0]] if hi else [])
        elif op == "v_permlane32_swap_b32":
            op, a = f"{op}:{a[1]}", [a[0], a[0], a[1]]
        elif op == "buffer_store_byte":
            op, a = f"v_store_byte:{a[2]}", ["null", a[0], a[1]]
        out.append((op, a))
    return out, labels


PROG = _program()


class Wave8(P.Wave):
    def __init__(self, wave, memories):
        self.cfg, self.wave, self.mem = CFG, wave, memories
        self.prog, self.labels = PROG
        self.s, self.v, self.a = {}, {}, {}
        self.lds = np.zeros(160 * 1024, np.uint8)
        self.vm, self.lgkm = [], []
        self.vcc = None

    def vval(self, t):
        if t == "vcc":
            return self.vcc
        if t.startswith("|"):
            return super().vval(t.strip("|")) & np.uint32(0x7FFFFFFF)
        return super().vval(t)

    def vset(self, t, x):
        if t == "vcc":
            self.vcc = np.asarray(x, np.uint32)
        elif t != "null":
            super().vset(t, x)

    def valu(self, op, x):
        lo = np.arange(64) < 32
        if op.startswith("v_permlane32_swap_b32"):
            a, b = x
            self.vset(op.split(":")[1], np.concatenate((a[32:], b[32:])))
            return np.concatenate((a[:32], b[:32]))
        if op.startswith("v_store_byte"):
            data, voff = x
            for lane, at in enumerate(self.access(op.split(":", 1)[1], voff, 1)):
                if at:
                    assert lo[lane]
                    at[0].data[at[1]] = data[lane] & 0xFF
                    at[0].hits[at[1]] += 1
            self.vm.append(("store", ()))
            return None
        if op == "v_cvt_scalef32_pk_fp8_f32":
            power = np.exp2(-((x[2] >> 23).astype(np.float64) - 127))
            with np.errstate(all="ignore"):
                two = [_e4m3((_f(t).astype(np.float64) * power).astype(np.float32)) for t in x[:2]]
            word = two[0] | two[1] << 8
            return (x[3] & 0xFFFF) | word << 16 if len(x) == 4 else word
        if op == "v_mov_b32":
            return x[0]
        if op == "v_max_i32":
            return np.maximum(x[0].view(np.int32), x[1].view(np.int32)).view(np.uint32)
        if op == "v_cmp_ne_u32":
            return x[0] != x[1]
        if op == "v_cmp_gt_u32":
            return x[0] > x[1]
        if op == "v_cndmask_b32":
            return np.where(x[2] != 0, x[1], x[0])
        return P.Wave.valu(op, x)


def _run(tiles, values, bias, bias_v, G, N, K, M):
    item = 2 if bias == "bf16" else 4
    width, blk = N // 2, M + 20
    sc, sq = width + 8, N + 16
    raw = P._bf16(bias_v).astype(np.uint16) if bias == "bf16" else bias_v
    mems = [P.Memory(P.OUT, np.full(2 * M * sc, 0xAB, np.uint8)), P.Memory(PRE8, np.full(M * sq, 0xAB, np.uint8)),
            P.Memory(P.BIAS, raw.reshape(-1).view(np.uint8).copy()), P.Memory(SCALES, np.full(N // 32 * blk, 0xAB, np.uint8))]
    S = (K + 127) // 128
    lane = np.arange(64, dtype=np.uint32)
    for wave in range(4):
        wm, wn = wave & 1, wave >> 1
        w = Wave8(wave, mems)
        state = dict(c0=0, nis=0, vmt=0, q0=0, q1=0, q2=0, np=0)
        for n, (g, row0, rows, n0) in enumerate(tiles):
            nxt = tiles[n + 1] if n + 1 < len(tiles) else tiles[n]
            w.tile = values[n]
            ptr = dict(bLT=P.A + row0 * 2880, bRT=P.B + n0 * 2880, bLN=P.A + nxt[1] * 2880, bRN=P.B + nxt[3] * 2880,
                       cT=P.OUT + 2 * (row0 * sc + n0 // 2), zT=PRE8 + row0 * sq + n0,
                       b=P.BIAS + (g * N + n0 + 160 * wn) * item, xT=SCALES + (n0 // 32 + 5 * wn) * blk + row0)
            ops = dict(state)
            for k, p in ptr.items():
                ops[f"{k}_lo"], ops[f"{k}_hi"] = p & M32, p >> 32
            ops.update(lds_base=0, w1k=1024 * wave, klenT=K, recAT=(rows - 1) * 2880, recBT=319 * 2880,
                       klenN=K if n + 1 < len(tiles) else 0, recAN=(nxt[2] - 1) * 2880, recBN=319 * 2880,
                       crecT=(rows * sc - n0 // 2) * 2, cm2=2 * sc, alpha=int(_bits(P.ALPHA)),
                       sw_epi=(128 * wm * sc + 80 * wn) * 2, vboff=lane * np.uint32(4 * item),
                       brec=160 * item if bias else 0, bf32=int(bias != "bf16"), nslope=int(_bits(-P.SLOPE * 1.44269504)),
                       limit=int(_bits(P.LIMIT)), shift=int(_bits(P.SHIFT)), zrecT=rows * sq - n0, zm2=sq,
                       sw_z=128 * wm * sq + 160 * wn, xrows=rows, xstep=blk,
                       xoff=np.where(lane < 32, 128 * wm + lane, 0x7FFF0000).astype(np.uint32))
            for j in range(CFG.nl):
                ops[f"voffL{j}"] = lane
            for j in range(CFG.nr):
                ops[f"voffR{j}"] = lane
            for side, base in (("am", 0), ("bn", CFG.rhs_off)):
                for x in ("lo0", "lo1", "hi0", "hi1"):
                    ops[side + x] = np.full(64, base, np.uint32)
            w.run(ops)
            state = {k: ops[k] for k in state}
            state["c0"] = (state["c0"] + S) % 2
        assert state["np"] == 0 and state["nis"] == 0
    return mems, sc, sq, blk


def _check(tiles, values, bias, bias_v, G, N, K, M):
    mems, sc, sq, blk = _run(tiles, values, bias, bias_v, G, N, K, M)
    z, covered = np.zeros((M, N), np.float32), np.zeros((M, N), bool)
    b = bias_v if bias else np.zeros_like(bias_v)
    for (g, row0, rows, n0), t in zip(tiles, values):
        with np.errstate(all="ignore"):
            z[row0:row0 + rows, n0:n0 + 320] = (t[:rows].astype(np.float64) * P.ALPHA + b[g, n0:n0 + 320]).astype(np.float32)
        covered[row0:row0 + rows, n0:n0 + 320] = True
    codes, scales = (t.numpy() for t in omx.quantize(torch.from_numpy(z), "e4m3"))
    q = mems[1].data.reshape(M, sq)
    assert (mems[1].hits.reshape(M, sq) == np.pad(covered, ((0, 0), (0, sq - N)))).all()
    assert (q[:, :N] == codes)[covered].all()
    hits = mems[3].hits.reshape(N // 32, blk)
    cells = np.pad(covered[:, ::32].T, ((0, 0), (0, blk - M)))
    assert (hits == cells).all()
    assert (mems[3].data.reshape(N // 32, blk)[:, :M] == scales.T)[cells[:, :M]].all()
    with np.errstate(all="ignore"):
        ref = P._silu_gate(z[:, 0::2].astype(np.float64), z[:, 1::2].astype(np.float64))
    live = covered[:, ::2]
    assert (mems[0].hits.reshape(M, 2 * sc) == np.repeat(np.pad(live, ((0, 0), (0, sc - N // 2))), 2, 1)).all()
    got = P._bf16_value(mems[0].data.reshape(M, 2 * sc)[:, :N].reshape(-1)).reshape(ref.shape)
    fine = live & np.isfinite(ref)
    assert (np.abs(got - ref)[fine] <= 2.0 ** -8 * np.abs(ref[fine]) + 1e-5).all()


@pytest.mark.parametrize("K,bias", [(64, "f32"), (128, None), (320, "bf16"), (2880, "bf16")])
def test_tiles(K, bias):
    rng = np.random.default_rng(K)
    G, N, M = 2, 640, 300
    tiles = [(0, 0, 256, 0), (0, 0, 256, 320), (0, 256, 37, 320), (1, 293, 1, 0)]       # group, first row, rows, column
    values = (rng.normal(size=(len(tiles), 256, 320)) * 6 * np.exp2(rng.integers(-20, 3, size=(len(tiles), 1, 320)))).astype(np.float32)
    bias_v = rng.normal(size=(G, N)).astype(np.float32)
    if bias == "bf16":
        bias_v = _f(P._bf16(bias_v) << 16)
    _check(tiles, values, bias, bias_v, G, N, K, M)


def test_zeros_subnormals_infinities():
    values = np.random.default_rng(3).normal(size=(1, 256, 320)).astype(np.float32)
    values[0, :, 32:64] = 0
    values[0, 0::5, 64:96] *= 2.0 ** -126
    values[0, 1::5, 100] = np.inf
    values[0, 2::5, 150] = np.nan
    values[0, 3::5, 200] = 3e38
    for r, m in enumerate((1.75, 1.8125, 1.8125 - 2.0 ** -22, 1.9999999)):
        values[0, 4 + 8 * r, 224:256] = np.float32(2 * m)
    _check([(0, 0, 256, 0)], values, None, np.zeros((1, 320), np.float32), 1, 320, 64, 256)


def test_hazards_and_include():
    """Two instructions between a transcendental and its use, wait states around the lanes' exchange; the include lists the
    configuration."""
    prog, _ = P._program(CFG)
    for k, ((op, a), (op2, a2)) in enumerate(zip(prog, prog[1:])):
        if op in ("v_exp_f32", "v_rcp_f32"):
            assert a[0] not in a2[1:], (op, a, op2, a2)
        if op2 == "v_permlane32_swap_b32":
            assert op == "s_nop" and int(a[0]) >= 4 and prog[k + 2][0] == "s_nop"
    text = open(W.GEN_PATH.replace("gen_vark_wide.py", "vark_wide_asm.inc")).read()
    assert f"#define GGEMM_WIDE_NOPERANDS_{CFG.name} {len(CFG.operands)}" in text


@pytest.mark.parametrize("G,N,K,M,act,residual,rows", [
    (8, 1040, 3696, 14998, 3, 0, 192), (2, 1680, 2608, 9592, 2, 1, 192), (9, 1504, 1840, 11078, 2, 0, 192),
    (4, 2096, 2880, 20000, 3, 0, 192), (3, 2704, 1056, 813, 3, 1, 64), (7, 2048, 1424, 5003, 2, 1, 128),
])
def test_choice_counts_the_tiles_that_run(pkg, G, N, K, M, act, residual, rows):
    """With z in 8 bits the 512-thread kernel's tiles are 384 columns wide whatever N: launches on which it measured 14 to 40 %
    faster than the 128-row tiles that an estimate with 320 columns took, next to others that stay."""
    got = pkg.load_library().ggemm_mx_keep_tile_rows(G, N, K, K, K, N // 2 if act == 3 else N, N, act, residual, M, 256)
    assert got == rows
