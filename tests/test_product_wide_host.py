"""CPU checks of the wide tiles with an epilogue (the KECONFIGS of ggemm-asm_amd/csrc/gen_vark_wide.py,
persistent_wide.h), before any GPU launch.

The per-tile assembly runs lane by lane in numpy (scalar and vector instructions, LDS, buffer loads and stores with
their bounds; an MFMA leaves a value of its tile, row and column in its accumulators, LDS-DMA moves nothing), with the
HIP tile loop around it restated, for each of the four waves over a sequence of tiles. Checked: every element of C
and of the kept z is written once, by its own value; rows past a group's end and bytes outside the tensors are not
touched; loads have completed (counted vmcnt and lgkmcnt, in order) where their results are used; staging stays
inside the wave's part of the freed slot; only clobbered registers are written, accumulators by MFMAs alone.
"""
import re

import numpy as np
import pytest

import test_vark_wide_host as W

GEN = W.GEN
M32 = W.M32
CFGS = {c.name: c for c in GEN.KECONFIGS}
ALPHA, SLOPE, LIMIT, SHIFT = 0.5, 1.702, 7.0, 1.0


def _program(cfg):
    g = GEN.GenKE(cfg)
    g.tile()
    prog, labels = [], {}
    for line in g.lines:
        if line.endswith(":"):
            labels[line[:-1]] = len(prog)
        else:
            op, _, rest = line.partition(" ")
            prog.append((op, [x.strip() for x in rest.split(",")] if rest else []))
    return prog, labels


PROGS = {n: _program(c) for n, c in CFGS.items()}


def _f(x):
    return np.asarray(x, np.uint32).view(np.float32)


def _bits(x):
    return np.asarray(x, np.float32).view(np.uint32)


def _bf16(x):
    u = _bits(x).astype(np.uint64)
    return (((u + 0x7FFF + ((u >> 16) & 1)) >> 16) & 0xFFFF).astype(np.uint32)


class Memory:
    """A tensor at an address: bytes, and how often each was written."""

    def __init__(self, base, data):
        self.base, self.data, self.hits = base, data, np.zeros(data.size, np.int32)


class Wave:
    def __init__(self, cfg, wave, memories):
        self.cfg, self.wave, self.mem = cfg, wave, memories
        self.prog, self.labels = PROGS[cfg.name]
        self.s, self.v, self.a = {}, {}, {}
        self.lds = np.zeros(160 * 1024, np.uint8)
        self.vm, self.lgkm = [], []           # outstanding operations in order: (kind, what)

    # ---- operands
    def ref(self, t):
        if t.startswith("%"):
            name, kind = self.cfg.operands[int(t[1:])]
            return name, kind
        return None

    def sval(self, t):
        r = self.ref(t)
        if r:
            assert "s" in r[1], f"scalar use of {r}"
            return self.ops[r[0]] & M32
        if re.fullmatch(r"s\d+|m0", t):
            return self.s[t]
        return int(t, 0) & M32

    def sset(self, t, x):
        r = self.ref(t)
        if r:
            assert r[1] == "+s", r
            self.ops[r[0]] = x & M32
            return
        assert t == "m0" or int(t[1:]) in self.cfg.sgpr_clobber, t
        self.s[t] = x & M32

    def vval(self, t):
        """64 lanes of a source: a vector register or operand, a scalar, a literal."""
        r = self.ref(t)
        if r and r[1] == "v":
            return np.broadcast_to(np.asarray(self.ops[r[0]], np.uint32), 64)
        m = re.fullmatch(r"v(\d+)", t)
        if m:
            n = int(m.group(1))
            assert not any(k == "load" and n in regs for k, regs, *_ in self.vm + self.lgkm), f"v{n} still in flight"
            return self.v[n]
        if re.fullmatch(r"-?\d+\.\d+", t):
            return np.full(64, _bits(float(t)), np.uint32)
        return np.full(64, self.sval(t), np.uint32)

    def vset(self, t, x):
        n = int(re.fullmatch(r"v(\d+)", t).group(1))
        assert n in self.cfg.vgpr_clobber and n < self.cfg.vacc0, t
        self.v[n] = np.asarray(x, np.uint32)

    @staticmethod
    def regs(t):
        m = re.fullmatch(r"v\[(\d+):(\d+)\]|v(\d+)", t)
        return list(range(int(m.group(1)), int(m.group(2)) + 1)) if m.group(1) else [int(m.group(3))]

    def rsrc(self, quad):
        lo = int(re.match(r"s\[(\d+)", quad).group(1))
        w = [self.s[f"s{r}"] for r in range(lo, lo + 4)]
        assert w[1] >> 16 == 0 and w[3] == GEN.WORD3
        return w[0] | w[1] << 32, w[2]

    def access(self, quad, voff, lane_bytes):
        """(memory, byte index) for each lane inside num_records, None for the others."""
        base, nrec = self.rsrc(quad)
        out = []
        for o in voff.astype(np.int64):
            if o + lane_bytes > nrec:
                assert o >= nrec or nrec == 0, "an access across the end"
                out.append(None)
                continue
            hit = [m for m in self.mem if m.base <= base + o and base + o + lane_bytes <= m.base + m.data.size]
            assert len(hit) == 1, "an access outside the tensors"
            out.append((hit[0], int(base + o - hit[0].base)))
        return out

    # ---- one tile
    def run(self, ops):
        self.ops, scc, pc = ops, 0, 0
        self.staging = False
        s32 = lambda x: x - (1 << 32) if x & 0x80000000 else x  # noqa: E731
        while pc < len(self.prog):
            op, a = self.prog[pc]
            pc += 1
            if op in ("s_cbranch_scc0", "s_cbranch_scc1", "s_branch"):
                if op == "s_branch" or scc == int(op[-1]):
                    pc = self.labels[a[0]]
            elif op in ("s_nop", "s_barrier"):
                pass
            elif op == "s_waitcnt":
                kind, n = re.fullmatch(r"(vmcnt|lgkmcnt)\((\d+)\)", a[0]).groups()
                assert int(n) <= (63 if kind == "vmcnt" else 15)
                q = self.vm if kind == "vmcnt" else self.lgkm
                del q[:max(0, len(q) - int(n))]
            elif op.startswith("s_cmp_"):
                x, y = self.sval(a[0]), self.sval(a[1])
                scc = int({"s_cmp_eq_u32": x == y, "s_cmp_lt_u32": x < y, "s_cmp_ge_u32": x >= y}[op])
            elif op == "s_cselect_b32":
                self.sset(a[0], self.sval(a[1]) if scc else self.sval(a[2]))
            elif op == "s_mov_b32":
                self.sset(a[0], self.sval(a[1]))
            elif op.startswith("s_"):
                x, y = self.sval(a[1]), self.sval(a[2])
                r = {"s_add_u32": x + y, "s_addc_u32": x + y + scc, "s_sub_u32": x - y, "s_sub_i32": x - y,
                     "s_mul_i32": x * y, "s_and_b32": x & y, "s_xor_b32": x ^ y, "s_lshl_b32": x << (y & 31),
                     "s_lshr_b32": x >> (y & 31), "s_min_i32": min(s32(x), s32(y)), "s_max_i32": max(s32(x), s32(y)),
                     "s_min_u32": min(x, y)}[op]
                if op in ("s_add_u32", "s_addc_u32"):
                    scc = int(r > M32)
                elif op == "s_sub_u32":
                    scc = int(r < 0)
                self.sset(a[0], r)
            elif op.startswith("v_mfma"):
                for t in (a[1], a[2]):
                    for n in self.regs(t):
                        self.vval(f"v{n}")                    # operands have arrived
                kind, lo = a[0][0], int(re.search(r"\[(\d+)", a[0]).group(1))
                blk = lo // 16 if kind == "a" else 16 + (lo - self.cfg.vacc0) // 16
                i, j = divmod(blk, self.cfg.bn)
                lane = np.arange(64)
                for n in range(16):
                    row = 128 * (self.wave & 1) + 32 * i + lane % 32
                    col = 160 * (self.wave >> 1) + 32 * j + 8 * (n // 4) + 4 * (lane // 32) + n % 4
                    (self.a if kind == "a" else self.v)[lo + n] = _bits(self.tile[row, col])
            elif op == "buffer_load_dwordx4" and a[-1].endswith("lds"):
                self.rsrc(a[1])
                self.vm.append(("dma", (), self.s["m0"] // self.cfg.slot))
            elif op.startswith("buffer_load"):
                dst = self.regs(a[0])
                for n in dst:
                    assert n in self.cfg.vgpr_clobber
                    self.v[n] = np.zeros(64, np.uint32)
                for lane, at in enumerate(self.access(a[2], self.vval(a[1]), 4 * len(dst))):
                    if at:
                        w = at[0].data[at[1]:at[1] + 4 * len(dst)].view(np.uint32)
                        for n, x in zip(dst, w):
                            self.v[n] = self.v[n].copy()
                            self.v[n][lane] = x
                self.vm.append(("load", dst))
            elif op == "buffer_store_dwordx4":
                data = np.stack([self.vval(f"v{n}") for n in self.regs(a[0])], 1)
                for lane, at in enumerate(self.access(a[2], self.vval(a[1]), 16)):
                    if at:
                        m, o = at
                        m.data[o:o + 16] = data[lane].view(np.uint8)
                        m.hits[o:o + 16] += 1
                self.vm.append(("store", ()))
            elif op.startswith("ds_"):
                self.ds(op, a)
            elif op == "v_readfirstlane_b32":
                self.sset(a[0], int(self.vval(a[1])[0]))
            elif op == "v_accvgpr_read_b32":
                self.vset(a[0], self.a[int(a[1][1:])])
            else:
                x = [self.vval(t) for t in a[1:]]
                scal = {t for t in a[1:] if re.fullmatch(r"s\d+", t) or (self.ref(t) and "s" in self.ref(t)[1])}
                assert len(scal) <= 1, f"{op} reads two scalars"
                with np.errstate(all="ignore"):
                    self.vset(a[0], self.valu(op, x))
        assert not self.lgkm or all(k == "write" for k, *_ in self.lgkm)

    @staticmethod
    def valu(op, x):
        f = [_f(t) for t in x]
        u = [t.astype(np.uint64) for t in x]
        lane = np.arange(64, dtype=np.uint32)
        int_ops = {
            "v_mbcnt_lo_u32_b32": lambda: np.minimum(lane, 32), "v_mbcnt_hi_u32_b32": lambda: np.maximum(lane, 32) - 32 + x[1],
            "v_and_b32": lambda: x[0] & x[1], "v_add_u32": lambda: (u[0] + u[1]) & M32,
            "v_add3_u32": lambda: (u[0] + u[1] + u[2]) & M32, "v_lshlrev_b32": lambda: (u[1] << u[0]) & M32,
            "v_lshrrev_b32": lambda: u[1] >> u[0], "v_lshl_add_u32": lambda: ((u[0] << u[1]) + u[2]) & M32,
            "v_mul_u32_u24": lambda: (u[0] * u[1]) & M32, "v_mul_lo_u32": lambda: (u[0] * u[1]) & M32,
            "v_cvt_pk_bf16_f32": lambda: _bf16(f[0]) | _bf16(f[1]) << 16}
        if op in int_ops:
            return int_ops[op]().astype(np.uint32)
        return _bits({"v_fma_f32": lambda: (f[0].astype(np.float64) * f[1] + f[2]).astype(np.float32),
                      "v_mul_f32": lambda: f[0] * f[1], "v_add_f32": lambda: f[0] + f[1],
                      "v_minimum3_f32": lambda: np.minimum(np.minimum(f[0], f[1]), f[2]),
                      "v_maximum3_f32": lambda: np.maximum(np.maximum(f[0], f[1]), f[2]),
                      "v_exp_f32": lambda: np.exp2(f[0]), "v_rcp_f32": lambda: np.float32(1) / f[0]}[op]())

    def ds(self, op, a):
        write = "write" in op
        last, _, mod = a[-1].partition(" ")
        off = int(mod.split(":")[1]) if mod else 0
        reg_t, addr_t = (last, a[0]) if write else (a[0], last)
        width = {"b32": 4, "b64": 8, "b128": 16}[op.split("_")[-1]]
        regs = self.regs(reg_t)
        assert 4 * len(regs) == width and 0 <= off < 65536
        addr = self.vval(addr_t).astype(np.int64) + off
        operand = not write and (self.cfg.vop0 <= regs[0]) and not self.staging
        if operand:                                   # of an MFMA: its slot's loads have completed
            slot = int(addr[0]) // self.cfg.slot
            assert not any(k == "dma" and rest[0] == slot for k, _, *rest in self.vm), "a stage read before its loads"
        else:
            self.staging = True
            lo = self.ops["lds_base"] + self.s["s81"]      # the freed slot
            rows, bias = lo + 16384 * self.wave, lo + GEN.BIAS_OFF + 1024 * self.wave
            assert all(rows <= x and x + width <= rows + 16384 or bias <= x and x + width <= bias + 1024 for x in addr)
        assert (addr % width == 0).all()
        if write:
            data = np.stack([self.vval(f"v{n}") for n in regs], 1)
            for x, d in zip(addr, data):
                self.lds[x:x + width] = np.ascontiguousarray(d).view(np.uint8)
            self.lgkm.append(("write", ()))
        else:
            for n in regs:
                assert n in self.cfg.vgpr_clobber and n < self.cfg.vacc0
                assert not any(k == "load" and n in r for k, r, *_ in self.lgkm), "two LDS loads into one register"
            got = np.stack([self.lds[x:x + width].view(np.uint32) for x in addr])
            for k, n in enumerate(regs):
                self.v[n] = got[:, k].copy()
            self.lgkm.append(("load", regs))


A, B, OUT, PRE, BIAS = 0x7F0000000000, 0x7E0000000000, 0x7D0000000000, 0x7C0000000000, 0x7B0000000000


def _silu_gate(g, u):
    g, u = np.minimum(g, LIMIT), np.clip(u, -LIMIT, LIMIT)
    return g / (1 + np.exp(-SLOPE * g)) * (u + SHIFT)


def _bf16_value(raw):
    return _f(raw.view(np.uint16).astype(np.uint32) << 16).astype(np.float64)


# rows of each tile in turn, tiles' columns, K of one stage, of a half stage, of several with and without a half one
@pytest.mark.parametrize("name", list(CFGS))
@pytest.mark.parametrize("K,bias", [(64, "f32"), (128, None), (320, "bf16"), (512, "f32"), (2880, "bf16")])
def test_tiles(name, K, bias):
    cfg = CFGS[name]
    rng = np.random.default_rng(K)
    G, N = 2, 640
    tiles = [(0, 0, 256, 0), (0, 0, 256, 320), (0, 256, 37, 320), (1, 293, 1, 0)]       # group, first row, rows, column
    M, gated = 300, cfg.gate
    width = N // 2 if gated else N
    sc, sz = width + 8, N + 16
    values = rng.normal(size=(len(tiles), 256, 320)).astype(np.float32) * 6
    bias_v = rng.normal(size=(G, N)).astype(np.float32)
    if bias == "bf16":
        raw = _bf16(bias_v).astype(np.uint16)
        bias_v = _f(raw.astype(np.uint32) << 16)
    else:
        raw = bias_v
    mems = [Memory(OUT, np.full(2 * M * sc, 0xAB, np.uint8)), Memory(PRE, np.full(2 * M * sz, 0xAB, np.uint8)),
            Memory(BIAS, raw.reshape(-1).view(np.uint8).copy())]
    S = (K + 127) // 128
    lane = np.arange(64, dtype=np.uint32)
    for wave in range(4):
        wm, wn = wave & 1, wave >> 1
        w = Wave(cfg, wave, mems)
        state = dict(c0=0, nis=0, vmt=0, q0=0, q1=0, q2=0, np=0)
        for n, (g, row0, rows, n0) in enumerate(tiles):
            nxt = tiles[n + 1] if n + 1 < len(tiles) else tiles[n]
            w.tile = values[n]
            item = 2 if bias == "bf16" else 4
            c0n = n0 // 2 if gated else n0
            ptr = dict(bLT=A + row0 * 2880, bRT=B + n0 * 2880, bLN=A + nxt[1] * 2880, bRN=B + nxt[3] * 2880,
                       cT=OUT + 2 * (row0 * sc + c0n), zT=PRE + 2 * (row0 * sz + n0),
                       b=BIAS + (g * N + n0 + 160 * wn) * item)
            ops = dict(state)
            for k, p in ptr.items():
                ops[f"{k}_lo"], ops[f"{k}_hi"] = p & M32, p >> 32
            ops.update(lds_base=0, w1k=1024 * wave, klenT=K, recAT=(rows - 1) * 2880, recBT=319 * 2880,
                       klenN=K if n + 1 < len(tiles) else 0, recAN=(nxt[2] - 1) * 2880, recBN=319 * 2880,
                       crecT=(rows * sc - c0n) * 2, cm2=2 * sc, alpha=int(_bits(ALPHA)),
                       sw_epi=(128 * wm * sc + (80 if gated else 160) * wn) * 2, vboff=lane * np.uint32(4 * item),
                       brec=160 * item if bias else 0, bf32=int(bias != "bf16"), nslope=int(_bits(-SLOPE * 1.44269504)),
                       limit=int(_bits(LIMIT)), shift=int(_bits(SHIFT)), zrecT=(rows * sz - n0) * 2, zm2=2 * sz,
                       sw_z=(128 * wm * sz + 160 * wn) * 2)
            for j in range(cfg.nl):
                ops[f"voffL{j}"] = lane
            for j in range(cfg.nr):
                ops[f"voffR{j}"] = lane
            for side, base in (("am", 0), ("bn", cfg.rhs_off)):
                for x in ("lo0", "lo1", "hi0", "hi1"):
                    ops[side + x] = np.full(64, base, np.uint32)
            w.run(ops)
            state = {k: ops[k] for k in state}
            state["c0"] = (state["c0"] + S) % 2
        assert state["np"] == 0 and state["nis"] == 0
    z = np.zeros((M, N))
    covered = np.zeros((M, N), bool)
    for (g, row0, rows, n0), t in zip(tiles, values):
        z[row0:row0 + rows, n0:n0 + 320] = ALPHA * t[:rows].astype(np.float64) + (bias_v[g, n0:n0 + 320] if bias else 0.0)
        covered[row0:row0 + rows, n0:n0 + 320] = True
    ref = _silu_gate(z[:, 0::2], z[:, 1::2]) if gated else z
    live = covered[:, ::2] if gated else covered
    for mem, stride, want, on in ((mems[0], sc, ref, live),) + (((mems[1], sz, z, covered),) if name.endswith("keep") else ()):
        hits = mem.hits.reshape(M, 2 * stride)
        cells = np.repeat(np.pad(on, ((0, 0), (0, stride - on.shape[1]))), 2, 1)
        assert (hits == cells).all()
        got = _bf16_value(mem.data.reshape(M, 2 * stride)[:, :2 * on.shape[1]].reshape(-1)).reshape(on.shape)
        assert (np.abs(got - want)[on] <= 2.0 ** -8 * np.abs(want[on]) + 1e-5).all()
    if not name.endswith("keep"):
        assert not mems[1].hits.any()


@pytest.mark.parametrize("name", list(CFGS))
def test_transcendental_results_are_read_two_instructions_later(name):
    """Their results need one wait state: the next instruction is another lane of work."""
    prog, _ = PROGS[name]
    for (op, a), (op2, a2) in zip(prog, prog[1:]):
        if op in ("v_exp_f32", "v_rcp_f32"):
            assert a[0] not in a2[1:], (op, a, op2, a2)


def test_generated_include_lists_the_configurations():
    text = open(W.GEN_PATH.replace("gen_vark_wide.py", "vark_wide_asm.inc")).read()
    for c in GEN.KECONFIGS:
        assert f"#define GGEMM_WIDE_NOPERANDS_{c.name} {len(c.operands)}" in text


@pytest.mark.parametrize("name", [c.name for c in GEN.KECONFIGS if c.gate])
def test_a_gate_far_below_zero_gives_zero(name):
    """Gates near the lowest finite value, whose product with the up half overflows, times a sigmoid of exactly zero:
    the result is the formula's zero, not NaN. One tile without a bias, z = alpha times its values."""
    cfg = CFGS[name]
    width, sc, sz, K = 160, 168, 328, 64
    tile = np.random.default_rng(1).normal(size=(256, 320)).astype(np.float32) * 6
    tile[::3, 0::4] = -3.3e38
    tile[1::3, 2::4] = -1e37
    tile[2::3, 0::8] = -400.0
    mems = [Memory(OUT, np.full(2 * 256 * sc, 0xAB, np.uint8)), Memory(PRE, np.full(2 * 256 * sz, 0xAB, np.uint8)),
            Memory(BIAS, np.zeros(16, np.uint8))]
    lane = np.arange(64, dtype=np.uint32)
    for wave in range(4):
        wm, wn = wave & 1, wave >> 1
        w = Wave(cfg, wave, mems)
        w.tile = tile
        ops = dict(c0=0, nis=0, vmt=0, q0=0, q1=0, q2=0, np=0)
        for k, p in dict(bLT=A, bRT=B, bLN=A, bRN=B, cT=OUT, zT=PRE, b=BIAS).items():
            ops[f"{k}_lo"], ops[f"{k}_hi"] = p & M32, p >> 32
        ops.update(lds_base=0, w1k=1024 * wave, klenT=K, recAT=255 * 2880, recBT=319 * 2880, klenN=0, recAN=255 * 2880,
                   recBN=319 * 2880, crecT=256 * sc * 2, cm2=2 * sc, alpha=int(_bits(ALPHA)),
                   sw_epi=(128 * wm * sc + 80 * wn) * 2, vboff=lane * np.uint32(16), brec=0, bf32=1,
                   nslope=int(_bits(-SLOPE * 1.44269504)), limit=int(_bits(LIMIT)), shift=int(_bits(SHIFT)),
                   zrecT=256 * sz * 2, zm2=2 * sz, sw_z=(128 * wm * sz + 160 * wn) * 2)
        ops.update({f"voffL{j}": lane for j in range(cfg.nl)})
        ops.update({f"voffR{j}": lane for j in range(cfg.nr)})
        for side, base in (("am", 0), ("bn", cfg.rhs_off)):
            ops.update({side + x: np.full(64, base, np.uint32) for x in ("lo0", "lo1", "hi0", "hi1")})
        w.run(ops)
    z = ALPHA * tile.astype(np.float64)
    with np.errstate(over="ignore"):
        want = _silu_gate(z[:, 0::2], z[:, 1::2])
    got = _bf16_value(mems[0].data.reshape(256, 2 * sc)[:, :2 * width].reshape(-1)).reshape(want.shape)
    assert not np.isnan(got).any()
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 1e-5).all()
