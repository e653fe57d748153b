"""The timed cases of what an MoE layer does around its expert products, and of those products with their epilogue.

A case names one operator (``op``) with its sizes and options:

* ``route``    -- ``route_experts``: router logits [T, E] to the k experts of each token and their weights; with
  ``grad`` the logits' gradient too
* ``dispatch`` -- ``plan_dispatch`` and ``dispatch_tokens``: the tokens' rows copied into expert order, the group
  offsets that the grouped products take
* ``combine``  -- ``combine_tokens``: each token's sum over its experts' rows by weight, with the residual stream
* ``exchange`` -- both ways in training: dispatch and combine, forward and backward
* ``product``  -- ``grouped_gemm_fp8_bias_act``: the grouped FP8 product with bias, activation and residual in its
  epilogue; with ``keep`` the value before the activation too, which the backward pass reads
* ``act_grad`` -- ``bias_act_backward``: the gradient of bias and activation, with the bias' gradient for each expert

2880 and 5760 are the feature sizes of the repository's own workloads, 32 experts and 131072 rows its full size.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DT = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
FMAX = 448.0
LINE = 128            # bytes of a cache line: the row alignment of the fp8 operands
NONE = -math.inf


def listed():
    return [
        # one token decoded: a launch and its host path
        {"name": "route one token", "op": "route", "T": 1, "E": 32, "k": 4, "dtype": "f32", "score": "softmax",
         "bias": False, "groups": 1, "top_groups": 1, "renorm": True, "scale": 1.0, "padded": 0, "grad": False},
        # a batch of prompts at the repository's expert count, some of its tokens padding (all experts masked)
        {"name": "route prompt", "op": "route", "T": 131072, "E": 32, "k": 4, "dtype": "bf16", "score": "softmax",
         "bias": False, "groups": 1, "top_groups": 1, "renorm": True, "scale": 1.0, "padded": 1000, "grad": False},
        # a training step of a router with sigmoid scores, balanced by a bias, experts taken from 4 of 8 groups
        {"name": "route train grouped", "op": "route", "T": 16384, "E": 256, "k": 8, "dtype": "f32",
         "score": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "renorm": True, "scale": 2.5, "padded": 0,
         "grad": True},
        # a decoding step of a small batch
        {"name": "dispatch decode", "op": "dispatch", "T": 16, "k": 4, "G": 32, "H": 2880, "dtype": "e4m3", "dropped": 0},
        # a batch of prompts, quantized once and copied to its experts: the repository's 131072 rows
        {"name": "dispatch prompt", "op": "dispatch", "T": 32768, "k": 4, "G": 32, "H": 2880, "dtype": "e4m3", "dropped": 0},
        # and back, into the residual stream
        {"name": "combine prompt", "op": "combine", "T": 32768, "k": 4, "G": 32, "H": 2880, "dtype": "bf16",
         "dropped": 0, "residual": True},
        # a training micro-batch of odd sizes with tokens dropped by the routing
        {"name": "exchange train ragged", "op": "exchange", "T": 5003, "k": 6, "G": 60, "H": 1424, "dtype": "bf16",
         "dropped": 150, "residual": True},
        # the gate and up product of one token's four experts: their weights are what is read
        {"name": "product one token", "op": "product", "G": 32, "M": 4, "n": 5760, "k": 2880, "lens": "single",
         "act": "swiglu", "bias": "bf16", "residual": False, "keep": False},
        # a decoding step of 64 tokens: a handful of rows for each expert
        {"name": "product decode", "op": "product", "G": 32, "M": 256, "n": 5760, "k": 2880, "lens": "even",
         "act": "swiglu", "bias": "bf16", "residual": False, "keep": False},
        # the forward pass of a full training micro-batch, with what its backward pass needs
        {"name": "product train full", "op": "product", "G": 32, "M": 131072, "n": 5760, "k": 2880, "lens": "even",
         "act": "swiglu", "bias": "f32", "residual": False, "keep": True},
        # feature sizes off the tiles' grid, skewed groups, an ungated activation added to a residual
        {"name": "product ragged", "op": "product", "G": 7, "M": 5003, "n": 2048, "k": 1424, "lens": "skew",
         "act": "gelu", "bias": "f32", "residual": True, "keep": False},
        # the gradient through bias and activation of the full micro-batch
        {"name": "activation gradient full", "op": "act_grad", "G": 32, "M": 131072, "n": 5760, "lens": "even",
         "act": "swiglu"},
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
    op = rng.choice(("route", "route", "dispatch", "combine", "exchange", "product", "product", "act_grad"))
    c = {"op": op}
    if op == "route":
        c["T"] = _log_int(rng, 1, 131072)
        c["groups"] = rng.choice((1, 1, 4, 8))
        c["E"] = c["groups"] * _log_int(rng, 2 if c["groups"] > 1 else 4, 256 // c["groups"])
        c["top_groups"] = rng.randint(1, c["groups"])
        c["k"] = _log_int(rng, 1, min(16, c["E"]))
        c["dtype"] = rng.choice(("bf16", "f32"))
        c["score"] = rng.choice(("softmax", "sigmoid"))
        c["bias"] = rng.random() < 0.5
        c["renorm"] = rng.random() < 0.7
        c["scale"] = rng.choice((1.0, 2.5))
        c["padded"] = rng.choice((0, c["T"] // 50))
        c["grad"] = rng.random() < 0.5
        return c
    if op in ("dispatch", "combine", "exchange"):
        c["G"] = _log_int(rng, 2, 256)
        c["k"] = _log_int(rng, 1, min(8, c["G"]))
        c["T"] = _log_int(rng, 1, 131072 // c["k"])
        c["H"] = _features(rng, 2880, 16 if op == "dispatch" else 8)
        c["dtype"] = rng.choice(("e4m3", "bf16")) if op == "dispatch" else rng.choice(("bf16", "bf16", "f32"))
        c["dropped"] = rng.choice((0, c["T"] * c["k"] // 30))
        if op != "dispatch":
            c["residual"] = rng.random() < 0.5
        return c
    c["G"], c["M"] = _log_int(rng, 1, 32), _log_int(rng, 1, 131072)
    c["n"] = _features(rng, 5760)
    c["lens"] = rng.choice(("even", "skew"))
    if op == "product":
        c["k"] = _features(rng, 2880)
        c["act"] = rng.choice(("swiglu", "swiglu", "silu", "gelu", "none"))
        c["bias"] = rng.choice(("none", "bf16", "f32"))
        c["residual"] = rng.random() < 0.4
        c["keep"] = rng.random() < 0.5
    else:
        c["act"] = rng.choice(("swiglu", "swiglu", "silu", "gelu"))
    return c


# --------------------------------------------------------------------------- inputs

# The gated activation's options: its sigmoid's slope, the clamp of both halves, what is added to the up half.
GATE = {"slope": 1.702, "limit": 7.0, "shift": 1.0}


def _gens(seed):
    return torch.Generator().manual_seed(seed), torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, std, dtype, gen):
    return (torch.randn(shape, device="cuda", generator=gen) * std).to(dtype)


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


def _fp8(shape, std, gen):
    """An e4m3 operand with its per-tensor scale, its rows on 128-byte lines."""
    x = _randn(shape, std, torch.float32, gen)
    scale = (x.abs().max().double() / FMAX).float()
    q = (x / scale).clamp_(-FMAX, FMAX).to(torch.float8_e4m3fn)
    wide = torch.zeros(tuple(shape[:-1]) + (-(-shape[-1] // LINE) * LINE,), dtype=torch.uint8, device="cuda")
    wide[..., :shape[-1]] = q.view(torch.uint8)
    return wide.view(q.dtype)[..., :shape[-1]], scale


def _keys64(case, logits, bias):
    """What the experts are chosen by, in 64 bits, with the scores."""
    x = logits.double()
    p = torch.softmax(x, 1) if case["score"] == "softmax" else torch.sigmoid(x)
    key = p if bias is None else p + bias.double()
    return (x if bias is None and case["groups"] == 1 else key).masked_fill(x == NONE, NONE), p


def _groups64(case, key):
    g = key.view(key.shape[0], case["groups"], -1)
    return g.topk(2, dim=2).values.sum(2)


def _choose64(case, key):
    if case["groups"] > 1:
        s = _groups64(case, key)
        best = s.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        keep = torch.zeros_like(s, dtype=torch.bool).scatter_(1, best, True)
        key = key.masked_fill(~keep.repeat_interleave(key.shape[1] // case["groups"], 1), NONE)
    return key.sort(dim=1, descending=True, stable=True)


def _unsettled(case, logits, bias):
    """Tokens whose choice hangs on the last bits of a score: two of the values that decide it differ, by less
    than what 32 bits resolve of them."""
    key, _ = _keys64(case, logits, bias)
    best = _choose64(case, key).values[:, :case["k"] + 1]
    gap = best[:, :-1] - best[:, 1:]
    bad = ((gap > 0) & (gap < 2e-5)).any(1)
    if case["groups"] > 1:
        s = _groups64(case, key).sort(dim=1, descending=True).values
        gap = (s[:, :-1] - s[:, 1:])[:, case["top_groups"] - 1:case["top_groups"]]
        bad |= ((gap > 0) & (gap < 2e-5)).any(1)
    return bad


def _logits(case, gen):
    T, E = case["T"], case["E"]
    popular = torch.randn(E, device="cuda", generator=gen) * 0.7   # some experts are liked by most tokens
    bias = (torch.randn(E, device="cuda", generator=gen) * 0.05) if case["bias"] else None

    def some(n):
        return (torch.randn((n, E), device="cuda", generator=gen) * 1.5 + popular).to(DT[case["dtype"]])

    logits = some(T)
    if case["bias"] or case["groups"] > 1:          # without them the logits themselves are compared
        bad = _unsettled(case, logits, bias).nonzero().flatten()
        while bad.numel():
            logits[bad] = some(bad.numel())
            bad = bad[_unsettled(case, logits[bad], bias)]
    if case["padded"]:
        logits[torch.randperm(T, device="cuda", generator=gen)[:case["padded"]]] = NONE
    return logits, bias


def _experts(case, gen):
    """k distinct experts for each token, the first of them liked best; some choices dropped (-1)."""
    T, k, G = case["T"], case["k"], case["G"]
    liked = torch.randn(G, device="cuda", generator=gen) * 0.7
    e = (torch.randn((T, G), device="cuda", generator=gen) + liked).topk(k, dim=1).indices.int()
    if case["dropped"]:
        e.view(-1)[torch.randperm(T * k, device="cuda", generator=gen)[:case["dropped"]]] = -1
    return e


def _make(case, seed):
    cpu, gpu = _gens(seed)
    op = case["op"]
    s = {"case": case}
    if op == "route":
        s["logits"], s["bias"] = _logits(case, gpu)
        if case["grad"]:
            s["dweights"] = _randn((case["T"], case["k"]), 1.0, torch.float32, gpu)
        return s
    if op in ("dispatch", "combine", "exchange"):
        T, k, H, dt = case["T"], case["k"], case["H"], DT[case["dtype"]]
        s["experts"] = _experts(case, gpu)
        if op == "dispatch":
            s["x"] = _fp8((T, H), 1.0, gpu)[0] if case["dtype"] == "e4m3" else _randn((T, H), 1.0, dt, gpu)
            return s
        w = torch.rand((T, k), device="cuda", generator=gpu) + 0.1
        s["weights"] = w / w.sum(1, keepdim=True)
        s["y"] = _randn((T * k, H), 0.5, dt, gpu)
        s["residual"] = _randn((T, H), 1.0, dt, gpu) if case["residual"] else None
        if op == "exchange":
            s["x"] = _randn((T, H), 1.0, dt, gpu)
            s["drows"] = _randn((T * k, H), 1e-3, dt, gpu)
            s["dout"] = _randn((T, H), 1e-3, dt, gpu)
        # the plan of the same routing: made before the experts ran, in hand when their rows are combined
        offs, slots, _ = _plan(s["experts"], case["G"])
        s["offs"], s["slots"] = offs, slots
        return s
    s["host_offs"] = _offsets(case, cpu)
    s["offs"] = torch.tensor(s["host_offs"], dtype=torch.int64, device="cuda")
    M, n = case["M"], case["n"]
    n_out = n // 2 if case["act"] == "swiglu" else n
    if op == "act_grad":
        s["pre"] = _randn((M, n), 2.0, torch.bfloat16, gpu)
        s["dout"] = _randn((M, n_out), 1e-3, torch.bfloat16, gpu)
        return s
    s["a"], s["sa"] = _fp8((M, case["k"]), 1.0, gpu)
    s["b"], s["sb"] = _fp8((case["G"], n, case["k"]), 2.0 / math.sqrt(case["k"]), gpu)
    s["bias"] = _randn((case["G"], n), 0.5, DT[case["bias"]], gpu) if case["bias"] != "none" else None
    s["residual"] = _randn((M, n_out), 1.0, torch.bfloat16, gpu) if case["residual"] else None
    return s


def prepare(case, seed):
    s = _make(case, seed)
    if case["op"] == "route" and case["grad"]:
        s["logits"].requires_grad_()
    if case["op"] == "exchange":
        for t in (s["x"], s["y"], s["weights"]):
            t.requires_grad_()
    return s


# --------------------------------------------------------------------------- the plain forms

def _route_plain(case, logits, bias, dweights):
    x = logits.detach().float()
    if case["score"] == "softmax":
        m = x.amax(1, keepdim=True)
        e = torch.exp(x - torch.where(m == NONE, 0.0, m))
        p = e / e.sum(1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-x))
    # without a bias or groups the order of the scores is the order of the logits
    key = x if bias is None and case["groups"] == 1 else p if bias is None else p + bias
    key = torch.where(x == NONE, NONE, key)
    if case["groups"] > 1:
        g = key.view(key.shape[0], case["groups"], -1)
        two = g.sort(dim=2, descending=True).values[:, :, :2].sum(2)
        rank = two.sort(dim=1, descending=True, stable=True).indices.argsort(dim=1)
        key = torch.where((rank < case["top_groups"])[:, :, None], g, NONE).view(key.shape)
    val, idx = key.sort(dim=1, descending=True, stable=True)
    val, idx = val[:, :case["k"]], idx[:, :case["k"]]
    live = val > NONE
    ps = torch.where(live, p.gather(1, idx), 0.0)
    total = None
    if not case["renorm"]:
        q = ps
    elif case["score"] == "softmax":
        xs = torch.where(live, x.gather(1, idx), NONE)
        m = xs.amax(1, keepdim=True)
        e = torch.exp(xs - torch.where(m == NONE, 0.0, m))
        q = torch.where(live, e / e.sum(1, keepdim=True), 0.0)
    else:
        total = ps.sum(1, keepdim=True).clamp(min=1e-20)
        q = ps / total
    out = {"weights": q * case["scale"], "experts": torch.where(live, idx, -1).int()}
    if dweights is None:
        return out
    d = torch.where(live, dweights * case["scale"], 0.0)
    if case["renorm"]:
        d = d - (d * q).sum(1, keepdim=True)
    if case["score"] == "softmax" and case["renorm"]:
        dl = torch.zeros_like(x).scatter_(1, idx, d * q)
    elif case["score"] == "softmax":
        dl = torch.zeros_like(x).scatter_(1, idx, d * ps) - torch.nan_to_num(p) * (d * ps).sum(1, keepdim=True)
    else:
        d = d / total if case["renorm"] else d
        dl = torch.zeros_like(x).scatter_(1, idx, d * ps * (1 / (1 + torch.exp(x.gather(1, idx)))))
    return {**out, "dlogits": torch.where(x == NONE, 0.0, dl).to(logits.dtype)}


def _plan(experts, G):
    """(group offsets, row of each choice or -1, choices in row order): rows ordered by expert, then by token."""
    flat = experts.flatten().long()
    key = torch.where((flat >= 0) & (flat < G), flat, G)
    ordered, order = key.sort(stable=True)
    offs = torch.searchsorted(ordered, torch.arange(G + 1, device="cuda"))
    slots = torch.empty_like(order).scatter_(0, order, torch.arange(order.numel(), device="cuda"))
    return offs, torch.where(key < G, slots, -1).view(experts.shape).int(), order


def _dispatch_plain(x, k, offs, order):
    kept = torch.arange(order.numel(), device="cuda") < offs[-1]
    if x.dtype == torch.float8_e4m3fn:
        rows = x.view(torch.uint8)[order // k]
        return torch.where(kept[:, None], rows, 0).view(x.dtype)
    return torch.where(kept[:, None], x[order // k], 0.0)


def _rows_of(y, slots):
    return torch.where(slots[:, :, None] >= 0, y[slots.clamp(min=0).long()].float(), 0.0)


def _combine_plain(y, slots, weights, residual):
    out = (_rows_of(y, slots) * weights[:, :, None]).sum(1)
    return (out if residual is None else out + residual.float()).to(y.dtype)


def _exchange_plain(s):
    case, y, w, dout = s["case"], s["y"].detach(), s["weights"].detach(), s["dout"]
    offs, slots, order = _plan(s["experts"], case["G"])
    rows = _dispatch_plain(s["x"].detach(), case["k"], offs, order)
    out = _combine_plain(y, slots, w, s["residual"])
    dx = _rows_of(s["drows"], slots).sum(1).to(y.dtype)
    dweights = (_rows_of(y, slots) * dout[:, None, :].float()).sum(2)
    kept = torch.arange(order.numel(), device="cuda") < offs[-1]
    dy = w.flatten()[order][:, None] * dout[order // case["k"]].float()
    return {"rows": rows, "out": out, "dx": dx, "dweights": dweights, "dy": torch.where(kept[:, None], dy, 0.0).to(y.dtype)}


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


def _product_plain(s):
    case = s["case"]
    z = torch.empty((case["M"], case["n"]), device="cuda")
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
    return {"out": out, "pre": z.bfloat16()} if case["keep"] else {"out": out}


def _act_grad_plain(s):
    case = s["case"]
    dz = _act_grad(s["pre"].float(), s["dout"].float(), case["act"])
    dbias = torch.zeros((case["G"], case["n"]), device="cuda")
    for g, lo, hi in _spans(s["host_offs"]):
        dbias[g] = dz[lo:hi].sum(0)
    return {"dpre": dz.bfloat16(), "dbias": dbias}


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "route":
        return _route_plain(case, s["logits"], s["bias"], s.get("dweights"))
    if op == "dispatch":
        offs, slots, order = _plan(s["experts"], case["G"])
        return {"rows": _dispatch_plain(s["x"], case["k"], offs, order), "offs": offs, "slots": slots}
    if op == "combine":
        return {"out": _combine_plain(s["y"], s["slots"], s["weights"], s["residual"])}
    if op == "exchange":
        return _exchange_plain(s)
    return _product_plain(s) if op == "product" else _act_grad_plain(s)


# --------------------------------------------------------------------------- one pass

def run(s):
    if not own:
        return _plain(s)
    from __graft_entry__ import load_package
    ggemm = load_package()
    case = s["case"]
    op = case["op"]
    if op == "route":
        s["logits"].grad = None
        weights, experts = ggemm.route_experts(
            s["logits"], case["k"], score=case["score"], bias=s["bias"], num_groups=case["groups"],
            top_groups=case["top_groups"], renormalize=case["renorm"], scale=case["scale"])
        if not case["grad"]:
            return {"weights": weights, "experts": experts}
        weights.backward(s["dweights"])
        return {"weights": weights, "experts": experts, "dlogits": s["logits"].grad}
    if op == "dispatch":
        plan = ggemm.plan_dispatch(s["experts"], case["G"])
        rows = ggemm.dispatch_tokens(s["x"], plan, row_align=LINE if case["dtype"] == "e4m3" else None)
        return {"rows": rows, "offs": plan.group_offs, "slots": plan.slots}
    if op == "combine":
        plan = ggemm.DispatchPlan(s["offs"], s["slots"])
        return {"out": ggemm.combine_tokens(s["y"], plan, s["weights"], s["residual"])}
    if op == "exchange":
        s["x"].grad = s["y"].grad = s["weights"].grad = None
        plan = ggemm.plan_dispatch(s["experts"], case["G"])
        rows = ggemm.dispatch_tokens(s["x"], plan)
        out = ggemm.combine_tokens(s["y"], plan, s["weights"], s["residual"])
        out.backward(s["dout"])
        rows.backward(s["drows"])
        return {"rows": rows, "out": out, "dx": s["x"].grad, "dweights": s["weights"].grad, "dy": s["y"].grad}
    gate = GATE if case["act"] == "swiglu" else {}
    act = None if case["act"] == "none" else case["act"]
    if op == "product":
        got = ggemm.grouped_gemm_fp8_bias_act(s["a"], s["b"], s["sa"], s["sb"], s["offs"], s["bias"], act,
                                              s["residual"], keep_preact=case["keep"], **gate)
        return {"out": got[0], "pre": got[1]} if case["keep"] else {"out": got}
    dpre, dbias = ggemm.bias_act_backward(s["dout"], s["pre"], s["offs"], act, **gate)
    return {"dpre": dpre, "dbias": dbias}


# --------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    op = case["op"]
    item = {"bf16": 2, "f32": 4, "e4m3": 1}.get(case.get("dtype"), 2)
    if op == "route":
        T, E, k = case["T"], case["E"], case["k"]
        grad = T * E * item + T * k * 4 if case["grad"] else 0
        return {"bytes": T * E * item + T * k * 8 + (4 * E if case["bias"] else 0) + grad,
                "flops": T * E * (10 if case["grad"] else 5)}
    if op in ("dispatch", "combine", "exchange"):
        T, k, H = case["T"], case["k"], case["H"]
        kept = T * k - case["dropped"]
        plan = 8 * T * k + 8 * (case["G"] + 1)
        token, row = T * H * item, kept * H * item
        tail = case["dropped"] * H * item              # rows without a token are written as zeros
        res = token if case.get("residual") else 0
        if op == "dispatch":
            return {"bytes": plan + token + row + tail, "flops": 0}
        combine = row + token + res + 8 * T * k
        if op == "combine":
            return {"bytes": combine, "flops": 2 * kept * H}
        # forward: plan, dispatch, combine; backward: dx from the rows' gradient, dy and the weights' from dout
        return {"bytes": plan + token + row + tail + combine + (row + token) + (token + row + tail + 4 * T * k),
                "flops": 7 * kept * H}
    G, M, n = case["G"], case["M"], case["n"]
    n_out = n // 2 if case["act"] == "swiglu" else n
    if op == "act_grad":
        return {"bytes": 2 * M * (2 * n + n_out) + 4 * G * n, "flops": 12 * M * n_out}
    k, used = case["k"], min(G, M)                     # experts without a row need no weight
    bias = used * n * {"none": 0, "bf16": 2, "f32": 4}[case["bias"]]
    out = 2 * M * (n_out + (n if case["keep"] else 0) + (n_out if case["residual"] else 0))
    return {"bytes": M * k + used * n * k + bias + out, "flops": 2 * M * n * k}


# --------------------------------------------------------------------------- the same in 64 bits

def _route64(case, s):
    x = s["logits"]
    key, p = _keys64(case, x, s["bias"])
    p = torch.nan_to_num(p)
    ordered = _choose64(case, key)
    val, idx = ordered.values[:, :case["k"]], ordered.indices[:, :case["k"]]
    live = val > NONE
    dweights = s.get("dweights")
    with torch.enable_grad():
        leaf = x.double().masked_fill(x == NONE, -1e4).requires_grad_()   # stands in for -inf: a score of zero
        score = torch.softmax(leaf, 1) if case["score"] == "softmax" else torch.sigmoid(leaf)
        q = score.gather(1, idx) * live
        if case["renorm"]:
            q = q / q.sum(1, keepdim=True).clamp(min=1e-300)
        w = q * case["scale"]
        out = {"weights": w.detach(), "experts": torch.where(live, idx, -1).int()}
        if dweights is not None:
            (out["dlogits"],) = torch.autograd.grad(w, leaf, dweights.double())
            out["dlogits"] = out["dlogits"].masked_fill(x == NONE, 0.0)
    return out


def _exchange64(case, s):
    T, k, H, G = case["T"], case["k"], case["H"], case["G"]
    e = s["experts"].flatten().long()
    rank = torch.argsort(torch.where(e < 0, G, e) * (T * k) + torch.arange(T * k, device="cuda"))
    kept = rank[:T * k - case["dropped"]]              # the choices that have a row, in row order
    slots = torch.full((T * k,), -1, device="cuda", dtype=torch.long)
    slots[kept] = torch.arange(kept.numel(), device="cuda")
    offs = torch.cat((torch.zeros(1, dtype=torch.long, device="cuda"),
                      (e[:, None] == torch.arange(G, device="cuda")).sum(0).cumsum(0)))
    out = {}
    if case["op"] != "combine":
        x = s["x"].double()
        rows = torch.zeros((T * k, H), dtype=torch.float64, device="cuda")
        rows[:kept.numel()] = x[kept // k]
        out["rows"] = rows
    if case["op"] == "dispatch":
        return {**out, "offs": offs, "slots": slots.view(T, k).int()}
    n = kept.numel()
    y, w = s["y"].double()[:n], s["weights"].double().flatten()[kept][:, None]
    into = torch.zeros((T, H), dtype=torch.float64, device="cuda") if s["residual"] is None else s["residual"].double()
    out["out"] = into.index_add(0, kept // k, y * w)
    if case["op"] == "exchange":
        dout = s["dout"].double()[kept // k]
        out["dx"] = torch.zeros((T, H), dtype=torch.float64, device="cuda").index_add(0, kept // k, s["drows"].double()[:n])
        dw = torch.zeros(T * k, dtype=torch.float64, device="cuda")
        dw[kept] = (dout * y).sum(1)
        out["dweights"] = dw.view(T, k)
        dy = torch.zeros((T * k, H), dtype=torch.float64, device="cuda")
        dy[:n] = dout * w
        out["dy"] = dy
    return out


def _act64(z, act):
    if act == "swiglu":
        g, u = z[:, ::2].clamp(max=GATE["limit"]), z[:, 1::2].clamp(-GATE["limit"], GATE["limit"])
        return (u + GATE["shift"]) * g * torch.sigmoid(GATE["slope"] * g)
    return {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "none": lambda v: v}[act](z)


def exact(case, seed):
    s = _make(case, seed)
    op = case["op"]
    if op == "route":
        return _route64(case, s)
    if op in ("dispatch", "combine", "exchange"):
        return _exchange64(case, s)
    n, M = case["n"], case["M"]
    n_out = n // 2 if case["act"] == "swiglu" else n
    if op == "act_grad":
        dpre = torch.zeros((M, n), dtype=torch.float64, device="cuda")
        dbias = torch.zeros((case["G"], n), dtype=torch.float64, device="cuda")
        for g, lo, hi in _spans(s["host_offs"]):
            z = s["pre"][lo:hi].double().requires_grad_()
            with torch.enable_grad():
                (dpre[lo:hi],) = torch.autograd.grad(_act64(z, case["act"]), z, s["dout"][lo:hi].double())
            dbias[g] = dpre[lo:hi].sum(0)
        return {"dpre": dpre, "dbias": dbias}
    out = torch.zeros((M, n_out), dtype=torch.float64, device="cuda")
    pre = torch.zeros((M, n), dtype=torch.float64, device="cuda") if case["keep"] else None
    for g, lo, hi in _spans(s["host_offs"]):
        z = s["sa"].double() * s["sb"].double() * (s["a"][lo:hi].double() @ s["b"][g].double().t())
        if s["bias"] is not None:
            z += s["bias"][g].double()
        out[lo:hi] = _act64(z, case["act"])
        if case["keep"]:
            pre[lo:hi] = z
    if s["residual"] is not None:
        out += s["residual"].double()
    return {"out": out, "pre": pre} if case["keep"] else {"out": out}
