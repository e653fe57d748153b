"""The timed cases of microscaled (MX) storage around an MoE layer's products: blocks of 32 values along a row share a
power of two, the values are e2m1 (4 bits) or e4m3 (8 bits).

A case names one operator (``op``) with its sizes and options:

* ``mx``       -- ``quantize_mx`` and ``dequantize_mx``: rows to their blocks and back, as a weight is stored and an
  activation checkpoint is kept and restored
* ``product``  -- ``grouped_gemm_mx_bias_act``: the grouped product of e2m1 weights with e2m1 or e4m3 activations, with
  bias, activation and residual in its epilogue
* ``keep``     -- ``grouped_gemm_fp8_bias_act(keep_preact="mxfp8")``: the FP8 product of the training layer, with the
  value before the activation kept in 8 bits for the backward pass
* ``act_grad`` -- ``bias_act_backward`` from that checkpoint: the gradient of bias and activation

2880 and 5760 are the feature sizes of the repository's own workloads, 32 experts and 131072 rows its full size.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
LINE = 128            # bytes of a cache line: the row alignment of the operands
BLOCK = 32            # values that share a scale
EMAX = {"e2m1": 2, "e4m3": 8}               # exponent of the format's largest value
ROUNDS_UP = {"e2m1": 1.75, "e4m3": 1.8125}  # a block's largest mantissa from which its exponent is one more
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one token's activations, before the product of a decoding step
        {"name": "mx one token", "op": "mx", "rows": 1, "cols": 2880, "dtype": "bf16", "fmt": "e4m3"},
        # all experts' gate and up weights, stored in 4 bits
        {"name": "mx weights", "op": "mx", "rows": 184320, "cols": 2880, "dtype": "bf16", "fmt": "e2m1"},
        # fp32 rows of an odd size, whose last block is half as long
        {"name": "mx ragged", "op": "mx", "rows": 5003, "cols": 1424, "dtype": "f32", "fmt": "e2m1"},
        # the gate and up product of one token's four experts: their weights are what is read
        {"name": "product one token", "op": "product", "G": 32, "M": 4, "n": 5760, "k": 2880, "lens": "single",
         "a": "e4m3", "act": "swiglu", "bias": "bf16", "residual": False},
        # a decoding step of 64 tokens: a handful of rows for each expert
        {"name": "product decode", "op": "product", "G": 32, "M": 256, "n": 5760, "k": 2880, "lens": "even",
         "a": "e4m3", "act": "swiglu", "bias": "bf16", "residual": False},
        # a large batch of prompts through the gate and up product, activations in 4 bits too
        {"name": "product prompt", "op": "product", "G": 32, "M": 131072, "n": 5760, "k": 2880, "lens": "even",
         "a": "e2m1", "act": "swiglu", "bias": "bf16", "residual": False},
        # and a smaller one through the down product, activations in 8 bits
        {"name": "product down", "op": "product", "G": 32, "M": 32768, "n": 2880, "k": 2880, "lens": "skew",
         "a": "e4m3", "act": "none", "bias": "bf16", "residual": False},
        # feature sizes off the tiles' grid, skewed groups, an ungated activation added to a residual
        {"name": "product ragged", "op": "product", "G": 7, "M": 5003, "n": 2048, "k": 1440, "lens": "skew",
         "a": "e2m1", "act": "gelu", "bias": "f32", "residual": True},
        # the forward pass of a full training micro-batch, its checkpoint in 8 bits
        {"name": "keep full", "op": "keep", "G": 32, "M": 131072, "n": 5760, "k": 2880, "lens": "even",
         "act": "swiglu", "bias": "f32", "residual": False},
        # the same of odd sizes, an ungated activation and a residual
        {"name": "keep ragged", "op": "keep", "G": 7, "M": 5003, "n": 2048, "k": 1424, "lens": "skew",
         "act": "gelu", "bias": "f32", "residual": True},
        # the gradient through bias and activation of the full micro-batch
        {"name": "activation gradient full", "op": "act_grad", "G": 32, "M": 131072, "n": 5760, "lens": "even",
         "act": "swiglu"},
        # and of a small one, whose last block is half as long
        {"name": "activation gradient ragged", "op": "act_grad", "G": 7, "M": 5003, "n": 1424, "lens": "skew",
         "act": "silu"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _features(rng, most, step=16):
    """A feature size: one of the workloads' own, or any multiple of ``step``."""
    own_sizes = [s for s in (2880, 5760) if s <= most]
    if own_sizes and rng.random() < 0.4:
        return rng.choice(own_sizes)
    return step * _log_int(rng, max(1, 64 // step), most // step)


def draw(rng: random.Random):
    op = rng.choice(("mx", "mx", "product", "product", "product", "keep", "act_grad"))
    c = {"op": op}
    if op == "mx":
        c["rows"], c["cols"] = _log_int(rng, 1, 131072), _features(rng, 5760)
        c["dtype"], c["fmt"] = rng.choice(("bf16", "f32")), rng.choice(("e2m1", "e4m3"))
        return c
    c["G"], c["M"] = _log_int(rng, 1, 32), _log_int(rng, 1, 131072)
    c["n"] = _features(rng, 5760)
    c["lens"] = rng.choice(("even", "skew"))
    if op != "act_grad":
        c["k"] = _features(rng, 2880, BLOCK if op == "product" else 16)
        if op == "product":
            c["a"] = rng.choice(("e2m1", "e4m3"))
        c["act"] = rng.choice(("swiglu", "swiglu", "silu", "gelu") + (("none",) if op == "product" else ()))
        c["bias"] = rng.choice(("none", "bf16", "f32"))
        c["residual"] = rng.random() < 0.4
    else:
        c["act"] = rng.choice(("swiglu", "swiglu", "silu", "gelu"))
    return c


# --------------------------------------------------------------------------- the block format

# The gated activation's options: its sigmoid's slope, the clamp of both halves, what is added to the up half.
GATE = {"slope": 1.702, "limit": 7.0, "shift": 1.0}


def _blocks(x):
    """fp32 rows as blocks [.., cols / 32, 32], the last one filled up with zeros."""
    cols = x.shape[-1]
    if cols % BLOCK:
        x = torch.nn.functional.pad(x, (0, BLOCK - cols % BLOCK))
    return x.unflatten(-1, (-1, BLOCK))


def _exponents(amax, fmt):
    """The blocks' exponents: the smallest at which the largest value, rounded as though the format had no largest one,
    stays within it; zero for blocks of zeros."""
    m, e = torch.frexp(amax)                           # amax = m 2^e, m in [0.5, 1)
    x = e - 1 - EMAX[fmt] + (2 * m >= ROUNDS_UP[fmt])
    return torch.where(amax > 0, x.clamp(-127, 127), 0)


def _scaled(x, exponents):
    """x 2^exponents, the power in two factors that are normal numbers."""
    half = exponents // 2
    return torch.ldexp(torch.ldexp(x, half), exponents - half)


def _round_e2m1(v):
    """Nearest e2m1 values, ties to the even code."""
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign(torch.round(a / step) * step, v)


def _encode(x, fmt):
    """(values of the format, exponents + 127 as bytes) of fp32 rows: values [.., cols] as fp32 or e4m3."""
    b = _blocks(x)
    e = _exponents(b.abs().amax(-1), fmt)
    v = _scaled(b, -e[..., None])
    v = _round_e2m1(v) if fmt == "e2m1" else v.to(torch.float8_e4m3fn)
    return v.flatten(-2)[..., :x.shape[-1]], (e + 127).to(torch.uint8)


def _pack(values):
    """e2m1 values to bytes, the even column in the low half."""
    levels = torch.tensor(E2M1, device=values.device)
    code = torch.searchsorted(levels, values.abs().contiguous()).to(torch.uint8) | (torch.signbit(values).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _levels(q):
    """What the stored values stand for before their scales, in fp32."""
    if q.dtype != torch.uint8:
        return q.float()
    levels = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=q.device)
    return torch.stack((levels[(q & 15).int()], levels[(q >> 4).int()]), -1).flatten(-2)


def _decode(q, scales):
    """The stored rows in fp32."""
    v = _levels(q)
    return _scaled(_blocks(v), scales.int()[..., None] - 127).flatten(-2)[..., :v.shape[-1]]


# --------------------------------------------------------------------------- inputs

def _gens(seed):
    return torch.Generator().manual_seed(seed), torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, std, dtype, gen):
    return (torch.randn(shape, device="cuda", generator=gen) * std).to(dtype)


def _features_of(shape, std, dtype, gen):
    """Rows whose features differ in size, as a network's do: neighbouring blocks have other scales."""
    size = torch.exp(0.5 * torch.randn(shape[-1], device="cuda", generator=gen))
    return (torch.randn(shape, device="cuda", generator=gen) * (std * size)).to(dtype)


def _offsets(case, rng):
    """Group lengths of the case's rows, summed up: one row each for distinct experts, as many rows as an even
    choice gives, or exponentially distributed lengths."""
    G, M = case["G"], case["M"]
    if case["lens"] == "single":
        lens = torch.zeros(G, dtype=torch.long)
        lens[torch.randperm(G, generator=rng)[:M]] = 1
    elif case["lens"] == "even":
        lens = torch.bincount(torch.multinomial(torch.ones(G), M, replacement=True, generator=rng), minlength=G)
    else:
        w = torch.empty(G, dtype=torch.float64).exponential_(generator=rng)
        lens = (w / w.sum() * M).long()
        lens[-1] = M - int(lens[:-1].sum())
    return [0] + lens.cumsum(0).tolist()


def _aligned(t, to):
    """The same bytes, their rows on multiples of ``to`` bytes."""
    raw = t.view(torch.uint8)
    wide = torch.zeros(tuple(raw.shape[:-1]) + (-(-raw.shape[-1] // to) * to,), dtype=torch.uint8, device="cuda")
    wide[..., :raw.shape[-1]] = raw
    return wide[..., :raw.shape[-1]].view(t.dtype)


def _mx(x, fmt):
    """(stored values, scales) of fp32 rows, laid out as a program keeps them: values on 128-byte lines, scales on 16
    bytes."""
    v, s = _encode(x, fmt)
    return _aligned(_pack(v) if fmt == "e2m1" else v, LINE), _aligned(s, 16)


def _mx_weights(G, n, k, gen):
    parts = [_mx(_features_of((n, k), 2.0 / math.sqrt(k), torch.float32, gen), "e2m1") for _ in range(G)]
    q, s = (torch.stack([p[i].new_zeros((n, p[i].stride(0))) for p in parts]) for i in (0, 1))
    for g, (pq, ps) in enumerate(parts):
        q[g, :, :pq.shape[1]], s[g, :, :ps.shape[1]] = pq, ps
    return q[..., :k // 2], s[..., :k // BLOCK]


def _fp8(shape, std, gen):
    """An e4m3 operand with its per-tensor scale, its rows on 128-byte lines."""
    x = _randn(shape, std, torch.float32, gen)
    scale = (x.abs().max().double() / 448.0).float()
    return _aligned((x / scale).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn), LINE), scale


def _checkpoint(z):
    """(values, scales) of z in 8 bits as the product keeps them: a scale's neighbour in memory is the next row's."""
    q, s = _encode(z, "e4m3")
    M, nb = s.shape
    by_block = torch.zeros((nb, -(-M // 16) * 16), dtype=torch.uint8, device="cuda")
    by_block[:, :M] = s.t()
    return q.contiguous(), by_block.t()[:M]


def prepare(case, seed):
    cpu, gpu = _gens(seed)
    op = case["op"]
    s = {"case": case}
    if op == "mx":
        x = _features_of((case["rows"], case["cols"]), 1.0, DT[case["dtype"]], gpu)
        if case["rows"] > 8:
            x[case["rows"] // 2] = 0                   # a row of padding
        s["x"] = x
        return s
    s["host_offs"] = _offsets(case, cpu)
    s["offs"] = torch.tensor(s["host_offs"], dtype=torch.int64, device="cuda")
    M, n = case["M"], case["n"]
    n_out = n // 2 if case["act"] == "swiglu" else n
    if op == "act_grad":
        s["pre"] = _checkpoint(_randn((M, n), 2.0, torch.float32, gpu))
        s["dout"] = _randn((M, n_out), 1e-3, torch.bfloat16, gpu)
        return s
    if op == "product":
        s["a"] = _mx(_features_of((M, case["k"]), 1.0, torch.float32, gpu), case["a"])
        s["b"] = _mx_weights(case["G"], n, case["k"], gpu)
    else:
        s["a"], s["sa"] = _fp8((M, case["k"]), 1.0, gpu)
        s["b"], s["sb"] = _fp8((case["G"], n, case["k"]), 2.0 / math.sqrt(case["k"]), gpu)
    s["bias"] = _randn((case["G"], n), 0.5, DT[case["bias"]], gpu) if case["bias"] != "none" else None
    s["residual"] = _randn((M, n_out), 1.0, torch.bfloat16, gpu) if case["residual"] else None
    return s


# --------------------------------------------------------------------------- the plain forms

def _erf_half(x):
    return 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))


def _act(z, act):
    if act == "swiglu":
        g, u = z[:, 0::2].clamp(max=GATE["limit"]), z[:, 1::2].clamp(-GATE["limit"], GATE["limit"])
        return g / (1 + torch.exp(-GATE["slope"] * g)) * (u + GATE["shift"])
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z * _erf_half(z) if act == "gelu" else z


def _act_grad(z, d, act):
    if act == "swiglu":
        z0, z1 = z[:, 0::2], z[:, 1::2]
        g, u = z0.clamp(max=GATE["limit"]), z1.clamp(-GATE["limit"], GATE["limit"])
        sg = 1 / (1 + torch.exp(-GATE["slope"] * g))
        dg = d * (u + GATE["shift"]) * sg * (1 + GATE["slope"] * g * (1 - sg))
        dg = torch.where(z0 > GATE["limit"], 0.0, dg)
        du = torch.where(z1.abs() > GATE["limit"], 0.0, d * g * sg)
        return torch.stack((dg, du), 2).view(z.shape)
    if act == "silu":
        sg = 1 / (1 + torch.exp(-z))
        return d * sg * (1 + z * (1 - sg))
    return d * (_erf_half(z) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi))


def _spans(offs):
    return [(g, lo, hi) for g, (lo, hi) in enumerate(zip(offs, offs[1:])) if hi > lo]


def _mx_plain(s):
    case = s["case"]
    v, scales = _encode(s["x"].float(), case["fmt"])
    back = _scaled(_blocks(v.float()), scales.int()[..., None] - 127).flatten(-2)[..., :case["cols"]]
    return {"values": back.bfloat16(), "scales": scales}


def _product_plain(s):
    case = s["case"]
    z = torch.empty((case["M"], case["n"]), device="cuda")
    if case["op"] == "product":
        a = _decode(*s["a"])
        for g, lo, hi in _spans(s["host_offs"]):
            z[lo:hi] = a[lo:hi] @ _decode(s["b"][0][g], s["b"][1][g]).t()
    else:
        for g, lo, hi in _spans(s["host_offs"]):
            z[lo:hi] = s["a"][lo:hi].float() @ s["b"][g].float().t()
        z *= s["sa"] * s["sb"]
    if s["bias"] is not None:
        lens = torch.diff(s["offs"])
        z += torch.repeat_interleave(s["bias"].float(), lens, 0, output_size=case["M"])
    out = _act(z, case["act"])
    if s["residual"] is not None:
        out = out + s["residual"].float()
    out = out.bfloat16()
    if case["op"] == "product":
        return {"out": out}
    q, scales = _encode(z, "e4m3")
    return {"out": out, "kept": q, "kept_scales": scales.view(torch.float8_e8m0fnu)}


def _act_grad_plain(s):
    case = s["case"]
    dz = _act_grad(_decode(*s["pre"]), s["dout"].float(), case["act"])
    dbias = torch.zeros((case["G"], case["n"]), device="cuda")
    for g, lo, hi in _spans(s["host_offs"]):
        dbias[g] = dz[lo:hi].sum(0)
    return {"dpre": dz.bfloat16(), "dbias": dbias}


# --------------------------------------------------------------------------- one pass

def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return _mx_plain(s) if op == "mx" else _act_grad_plain(s) if op == "act_grad" else _product_plain(s)
    from __graft_entry__ import load_package
    ggemm = load_package()
    if op == "mx":
        kept = ggemm.quantize_mx(s["x"], case["fmt"])
        return {"values": ggemm.dequantize_mx(kept), "scales": kept.scales}
    act = None if case["act"] == "none" else case["act"]
    gate = GATE if act == "swiglu" else {}
    if op == "product":
        return {"out": ggemm.grouped_gemm_mx_bias_act(ggemm.MXTensor(*s["a"]), ggemm.MXTensor(*s["b"]), s["offs"],
                                                      s["bias"], act, s["residual"], **gate)}
    if op == "keep":
        out, kept = ggemm.grouped_gemm_fp8_bias_act(s["a"], s["b"], s["sa"], s["sb"], s["offs"], s["bias"], act,
                                                    s["residual"], keep_preact="mxfp8", **gate)
        return {"out": out, "kept": kept.q, "kept_scales": kept.scales.view(torch.float8_e8m0fnu)}
    dpre, dbias = ggemm.bias_act_backward(s["dout"], ggemm.MXTensor(*s["pre"]), s["offs"], act, **gate)
    return {"dpre": dpre, "dbias": dbias}


# --------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    op = case["op"]
    if op == "mx":
        rows, cols = case["rows"], case["cols"]
        stored = cols // (2 if case["fmt"] == "e2m1" else 1) + -(-cols // BLOCK)
        read = cols * (2 if case["dtype"] == "bf16" else 4)
        return {"bytes": rows * (read + 2 * stored + 2 * cols), "flops": 4 * rows * cols}
    G, M, n = case["G"], case["M"], case["n"]
    n_out = n // 2 if case["act"] == "swiglu" else n
    kept = M * (n + -(-n // BLOCK))
    if op == "act_grad":
        return {"bytes": kept + 2 * M * (n + n_out) + 4 * G * n, "flops": 12 * M * n_out}
    k, used = case["k"], min(G, M)                     # experts without a row need no weight
    bias = used * n * {"none": 0, "bf16": 2, "f32": 4}[case["bias"]]
    out = 2 * M * n_out * (2 if case["residual"] else 1)
    if op == "keep":
        return {"bytes": M * k + used * n * k + bias + out + kept, "flops": 2 * M * n * k}
    a = M * (k // (2 if case["a"] == "e2m1" else 1) + k // BLOCK)
    return {"bytes": a + used * n * (k // 2 + k // BLOCK) + bias + out, "flops": 2 * M * n * k}


# --------------------------------------------------------------------------- the same in 64 bits

def _decode64(q, scales):
    if q.dtype == torch.uint8:
        code = torch.stack((q % 16, q // 16), -1).flatten(-2).long()
        e, m, sign = code // 2 % 4, code % 2, 1.0 - 2.0 * (code // 8).double()
        v = sign * torch.where(e > 0, (1.0 + 0.5 * m) * 2.0 ** (e - 1).double(), 0.5 * m)
    else:
        v = q.double()
    power = torch.pow(2.0, scales.double() - 127).repeat_interleave(BLOCK, -1)[..., :v.shape[-1]]
    return v * power


def _mx64(case, x):
    fmt, x = case["fmt"], x.double()
    codes = (torch.arange(8) if fmt == "e2m1" else torch.arange(127)).to(torch.uint8)
    table = (torch.tensor(E2M1) if fmt == "e2m1" else codes.view(torch.float8_e4m3fn).float()).double().cuda()
    middle = (table[1:] + table[:-1]) / 2
    values, scales = torch.empty_like(x), []
    for c in range(0, case["cols"], BLOCK):
        b = x[:, c:c + BLOCK]
        top = b.abs().amax(1)
        e = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
        e = torch.where(torch.exp2(e) > torch.where(top > 0, top, 1.0), e - 1, e) - EMAX[fmt]
        past = 1.5 * table[-1] - 0.5 * table[-2]       # half a step past the largest value
        e = torch.where(top >= past * torch.exp2(e), e + 1, e)
        e = torch.where(top > 0, e, 0.0).clamp(-127, 127)
        v = (b.abs() / torch.exp2(e)[:, None]).contiguous()
        i = torch.bucketize(v, middle, right=True)     # a value on a middle belongs to the code above
        tie = (i > 0) & (v == middle[(i - 1).clamp(min=0)]) & (i % 2 == 1)
        values[:, c:c + BLOCK] = torch.sign(b) * table[i - tie.long()] * torch.exp2(e)[:, None]
        scales.append((e + 127).to(torch.uint8))
    return {"values": values, "scales": torch.stack(scales, 1)}


def _act64(z, act):
    if act == "swiglu":
        g, u = z[:, ::2].clamp(max=GATE["limit"]), z[:, 1::2].clamp(-GATE["limit"], GATE["limit"])
        return (u + GATE["shift"]) * g * torch.sigmoid(GATE["slope"] * g)
    return {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "none": lambda v: v}[act](z)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "mx":
        return _mx64(case, s["x"])
    n, M = case["n"], case["M"]
    n_out = n // 2 if case["act"] == "swiglu" else n
    if op == "act_grad":
        dpre = torch.zeros((M, n), dtype=torch.float64, device="cuda")
        dbias = torch.zeros((case["G"], n), dtype=torch.float64, device="cuda")
        for g, lo, hi in _spans(s["host_offs"]):
            z = _decode64(s["pre"][0][lo:hi], s["pre"][1][lo:hi]).requires_grad_()
            with torch.enable_grad():
                (dpre[lo:hi],) = torch.autograd.grad(_act64(z, case["act"]), z, s["dout"][lo:hi].double())
            dbias[g] = dpre[lo:hi].sum(0)
        return {"dpre": dpre, "dbias": dbias}
    out = torch.zeros((M, n_out), dtype=torch.float64, device="cuda")
    for g, lo, hi in _spans(s["host_offs"]):
        if op == "product":
            z = _decode64(s["a"][0][lo:hi], s["a"][1][lo:hi]) @ _decode64(s["b"][0][g], s["b"][1][g]).t()
        else:
            z = s["sa"].double() * s["sb"].double() * (s["a"][lo:hi].double() @ s["b"][g].double().t())
        if s["bias"] is not None:
            z += s["bias"][g].double()
        out[lo:hi] = _act64(z, case["act"])
    if s["residual"] is not None:
        out += s["residual"].double()
    return {"out": out} if op == "product" else {"out": out, "kept": None, "kept_scales": None}
