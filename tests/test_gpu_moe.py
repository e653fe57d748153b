"""Routing, dispatch and combination on the GPU against the 64-bit oracle, at the sizes and masks where they can go
wrong.

Tolerances. Weights and gradients of routing: expf of a difference of logits d has the relative error of the
difference's rounding, |d| 2^-24, beside a few roundings of exp, the sum (at most 4 + 6 additions deep) and the
divisions: (24 + range) 2^-23 covers them; gradients add the products' differences, taken against the largest term of
a token. Sums of rows: bf16 results are rounded once (2^-8 relative, half a unit of 8 bits) from an fp32 sum of k + 1 terms, each rounding
2^-24 of the sum of magnitudes.
"""
import numpy as np
import pytest
import torch

from oracle import moe_oracle as orm

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -23


def _np(t):
    return t.detach().cpu().double().numpy()


def _check_weights(w, ref, x, floor=1e-37):
    span = float(np.ptp(np.where(np.isfinite(x), x, 0.0))) if x.size else 0.0
    err = np.abs(w - ref)
    ok = (err <= (24 + span) * EPS * np.abs(ref) + floor) | (np.isnan(w) & np.isnan(ref))
    assert ok.all(), (err[~ok].max(), np.argwhere(~ok)[:3])


def _run(pkg, x, k, bias=None, **kw):
    w, e = pkg.route_experts(x, k, bias=bias, **kw)
    assert w.dtype == torch.float32 and e.dtype == torch.int32 and tuple(w.shape) == tuple(e.shape) == (x.shape[0], k)
    return _np(w), e.cpu().numpy()


# experts on both sides of every layout's edge, from one lane to sixteen per lane; k up to all of them
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("E,k,T", [(1, 1, 5), (2, 2, 1), (7, 7, 33), (8, 1, 1), (9, 4, 31), (16, 16, 100), (31, 4, 257),
                                   (32, 4, 1), (32, 32, 65), (33, 8, 40), (64, 6, 17), (65, 64, 9), (128, 8, 513),
                                   (129, 2, 3), (256, 8, 130), (257, 10, 5), (512, 22, 4), (513, 1, 7), (1000, 64, 3),
                                   (1024, 8, 6)])
@pytest.mark.parametrize("score,renorm,scale", [("softmax", True, 1.0), ("softmax", False, 2.5), ("sigmoid", True, 1.0),
                                                ("sigmoid", False, 0.5)])
def test_route_by_logit(pkg, dtype, E, k, T, score, renorm, scale):
    """Without bias and groups the choice is by the logits: exact, ties (bf16 has many) by the lower index."""
    gen = torch.Generator().manual_seed(E * 1000 + k)
    x = (torch.randn((T, E), generator=gen) * 2).to(dtype).cuda()
    w, e = _run(pkg, x, k, score=score, renormalize=renorm, scale=scale)
    rw, re, _ = orm.route(_np(x), k, score, renormalize=renorm, scale=scale)
    assert np.array_equal(e, re)
    _check_weights(w, rw, _np(x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("E,k,T,groups,top,best", [(32, 4, 70, 1, 1, 2), (8, 2, 33, 4, 2, 2), (64, 6, 40, 8, 3, 1),
                                                   (160, 6, 50, 8, 3, 2), (256, 8, 64, 8, 4, 2), (60, 5, 20, 20, 7, 2),
                                                   (96, 8, 20, 3, 1, 2), (1024, 16, 5, 32, 4, 2), (12, 6, 9, 12, 4, 1),
                                                   (256, 8, 31, 1, 1, 1), (24, 8, 21, 4, 1, 2)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_route_by_score_and_groups(pkg, dtype, E, k, T, groups, top, best, score, biased):
    gen = torch.Generator().manual_seed(E + k + groups)
    x = (torch.randn((T, E), generator=gen) * 2).to(dtype).cuda()
    bias = (torch.randn(E, generator=gen) * 0.1).cuda() if biased else None
    w, e = _run(pkg, x, k, bias=bias, score=score, num_groups=groups, top_groups=top, group_best=best)
    rw, re, margin = orm.route(_np(x), k, score, None if bias is None else _np(bias), groups, top, best)
    sure = margin > 2e-6                         # fp32 keys of order one: 2^-23 apart, a few roundings each
    assert sure.mean() > 0.7
    assert np.array_equal(e[sure], re[sure])
    _check_weights(w[sure], rw[sure], _np(x))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("biased", [False, True])
def test_route_masks_and_special_values(pkg, score, renorm, biased):
    """Masked experts, tokens with fewer experts left than k or none, the type's lowest value, infinities, NaN."""
    inf, low = float("inf"), torch.finfo(torch.float32).min
    x = torch.zeros((9, 40))
    x[:] = torch.linspace(-3, 3, 40)
    x[0] = -inf                                  # nothing left
    x[1, 1:] = -inf                              # one left
    x[2, ::2] = -inf
    x[3] = low                                   # the lowest finite value masks nothing
    x[4, 5] = inf
    x[5, 7] = float("nan")
    x[5, 3] = -inf
    x[6] = 0.0
    x[6, ::3] = -0.0                             # zeros of both signs are equal
    x[7] = 100.0
    x[8, :38] = -inf
    bias = torch.linspace(0.3, -0.3, 40)
    bias[39] = -inf if biased else 0.0
    b = bias.cuda() if biased else None
    w, e = _run(pkg, x.cuda(), 4, bias=b, score=score, renormalize=renorm)
    rw, re, _ = orm.route(x.numpy(), 4, score, bias.numpy() if biased else None, renormalize=renorm)
    assert np.array_equal(e, re)
    _check_weights(w[[0, 1, 2, 6, 7, 8]], rw[[0, 1, 2, 6, 7, 8]], x.numpy()[[0, 1, 2, 6, 7, 8]])
    for t in (3, 4, 5):
        np.testing.assert_array_equal(np.isnan(w[t]), np.isnan(rw[t]))
    assert np.allclose(w[3], rw[3], atol=1e-6)


def test_route_strides_and_empty(pkg):
    base = torch.randn((50, 100), generator=torch.Generator().manual_seed(1)).cuda()
    for view in (base[:, 3:36], base[::2, :33], base.t()[:, :30], base[:1, 5:38], base[0].expand(6, 100)):
        w, e = _run(pkg, view, 5)
        rw, re, _ = orm.route(_np(view), 5)
        assert np.array_equal(e, re)
        _check_weights(w, rw, _np(view))
    w, e = pkg.route_experts(base[:0], 5)
    assert tuple(w.shape) == (0, 5) and tuple(e.shape) == (0, 5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("E,k,T,groups,top", [(32, 4, 37, 1, 1), (8, 8, 5, 1, 1), (256, 8, 21, 8, 4), (60, 6, 3, 1, 1),
                                              (1000, 64, 2, 1, 1), (128, 1, 9, 4, 1), (24, 8, 11, 4, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_gradient(pkg, dtype, E, k, T, groups, top, score, renorm):
    gen = torch.Generator().manual_seed(E + k)
    x = (torch.randn((T, E), generator=gen) * 2).to(dtype).cuda()
    x[0, ::3] = -float("inf")
    if T > 2:
        x[2] = -float("inf")
    d = torch.randn((T, k), generator=gen).cuda()
    leaf = x.clone().requires_grad_()
    w, e = pkg.route_experts(leaf, k, score=score, renormalize=renorm, num_groups=groups, top_groups=top, scale=1.5)
    assert not e.requires_grad
    w.backward(d)
    plain, _ = pkg.route_experts(x, k, score=score, renormalize=renorm, num_groups=groups, top_groups=top, scale=1.5)
    assert torch.equal(plain, w)
    assert leaf.grad.dtype == dtype
    got, en = _np(leaf.grad), e.cpu().numpy()
    ref = orm.route_backward(_np(d), _np(x), en, score, renorm, 1.5)
    # terms of a token's gradient: |d| scale times weights of at most one
    size = 1.5 * np.abs(_np(d)).sum(1, keepdims=True)
    tol = 40 * EPS * size + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0) * np.abs(ref)
    assert (np.abs(got - ref) <= tol).all(), np.abs(got - ref).max()


@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route_gradient_against_differences(pkg, score, renorm):
    """dlogits against central differences of the oracle's weights, h^2 of which is 1e-8."""
    gen = torch.Generator().manual_seed(7)
    x, d = torch.randn((6, 16), generator=gen), torch.randn((6, 3), generator=gen)
    leaf = x.cuda().requires_grad_()
    w, e = pkg.route_experts(leaf, 3, score=score, renormalize=renorm)
    w.backward(d.cuda())
    e, h = e.cpu().numpy().astype(np.int64), 1e-4
    for i in range(16):
        up, dn = x.double().numpy().copy(), x.double().numpy().copy()
        up[:, i] += h
        dn[:, i] -= h
        diff = orm.weights_of(up, e, score, renorm, 1.0) - orm.weights_of(dn, e, score, renorm, 1.0)
        np.testing.assert_allclose(_np(leaf.grad)[:, i], (diff * d.numpy()).sum(1) / (2 * h), atol=2e-6)


# --------------------------------------------------------------------------- the order

# one workgroup, its edge, several; one choice and none; experts on both sides of a power of two; all in one expert
@pytest.mark.parametrize("T,k,G", [(0, 2, 4), (1, 1, 1), (1, 4, 32), (64, 1, 2), (65, 3, 7), (256, 8, 8), (512, 4, 33),
                                   (683, 3, 60), (2048, 1, 255), (2049, 1, 256), (5000, 6, 64), (4097, 2, 2047),
                                   (40000, 8, 128), (70000, 2, 3)])
@pytest.mark.parametrize("kind", ["even", "one", "dropped"])
def test_plan(pkg, T, k, G, kind):
    gen = torch.Generator().manual_seed(T + G)
    e = torch.randint(0, G, (T, k), generator=gen, dtype=torch.int32)
    if kind == "one":
        e[:] = G - 1
    if kind == "dropped":
        e[torch.rand((T, k), generator=gen) < 0.3] = -1
        e[torch.rand((T, k), generator=gen) < 0.1] = G          # another rank's expert
    plan = pkg.plan_dispatch(e.cuda(), G)
    offs, slots = orm.plan(e.numpy(), G)
    assert np.array_equal(plan.group_offs.cpu().numpy(), offs)
    assert np.array_equal(plan.slots.cpu().numpy(), slots)
    again = pkg.plan_dispatch(e.cuda(), G)
    assert torch.equal(again.slots, plan.slots)


def _some_plan(pkg, T, k, G, dropped, seed=0):
    gen = torch.Generator().manual_seed(seed + T)
    e = torch.randint(0, G, (T, k), generator=gen, dtype=torch.int32)
    if dropped:
        e[torch.rand((T, k), generator=gen) < dropped] = -1
    return pkg.plan_dispatch(e.cuda(), G), gen


# rows of whole 16-byte words, of 4- and 2-byte ones and of single bytes; longer than a wave's step, shorter than a lane
SIZES = [(1, 1, 1, 8, 0.0), (1, 4, 32, 2880, 0.0), (37, 3, 5, 1024, 0.2), (130, 2, 7, 33, 0.2), (300, 8, 16, 1000, 0.5),
         (5, 1, 3, 5001, 1.0), (64, 4, 8, 4096, 0.0), (9, 5, 4, 1, 0.3), (1000, 6, 60, 72, 0.1)]


@pytest.mark.parametrize("T,k,G,H,dropped", SIZES)
@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.uint8, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("align", [None, 128])
def test_dispatch(pkg, T, k, G, H, dropped, dtype, align):
    plan, gen = _some_plan(pkg, T, k, G, dropped)
    wide = torch.randint(0, 127, (T, H + 3, 4), generator=gen, dtype=torch.uint8)
    item = torch.empty(0, dtype=dtype).element_size()
    base = wide[:, :, :item].contiguous().view(dtype).reshape(T, H + 3).cuda()
    for x in (base[:, :H].contiguous(), base[:, 2:2 + H]):
        rows = pkg.dispatch_tokens(x, plan, row_align=align)
        assert tuple(rows.shape) == (T * k, H) and rows.dtype == dtype
        if align:
            assert rows.stride(0) * item % align == 0 and rows.data_ptr() % align == 0
        got = rows.contiguous().view(torch.uint8).reshape(T * k, H * item).cpu()
        src = x.contiguous().view(torch.uint8).reshape(T, H * item).cpu()
        ref = torch.zeros((T * k, H * item), dtype=torch.uint8)
        slots = plan.slots.cpu().long()
        for j in range(k):
            live = slots[:, j] >= 0
            ref[slots[live, j]] = src[live]
        assert torch.equal(got, ref)


def _rows_ref(y, slots):
    out = np.zeros((*slots.shape, y.shape[1]))
    out[slots >= 0] = y[slots[slots >= 0]]
    return out


@pytest.mark.parametrize("T,k,G,H,dropped", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("weighted,residual", [(True, True), (True, False), (False, True), (False, False)])
def test_combine_and_its_gradients(pkg, T, k, G, H, dropped, dtype, weighted, residual):
    plan, gen = _some_plan(pkg, T, k, G, dropped)
    M = T * k
    y = torch.randn((M, H + 1), generator=gen).to(dtype).cuda()[:, 1:] if H % 2 else \
        torch.randn((M, H), generator=gen).to(dtype).cuda()
    kept = int(plan.group_offs[-1])
    y[kept:] = float("nan")                              # rows without a choice are never read
    w = torch.randn((T, k), generator=gen).cuda() if weighted else None
    r = torch.randn((T, H), generator=gen).to(dtype).cuda() if residual else None
    dout = torch.randn((T, H), generator=gen).to(dtype).cuda()
    leaves = [None if t is None else t.detach().requires_grad_() for t in (y, w, r)]
    out = pkg.combine_tokens(leaves[0], plan, leaves[1], leaves[2])
    assert out.dtype == dtype and torch.equal(out, pkg.combine_tokens(y, plan, w, r))
    out.backward(dout)
    slots = plan.slots.cpu().numpy()
    rows, wn = _rows_ref(_np(y), slots), np.ones((T, k)) if w is None else _np(w)
    terms = rows * np.where(slots >= 0, wn, 0.0)[:, :, None]
    ref = terms.sum(1) + (0.0 if r is None else _np(r))
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    size = np.abs(terms).sum(1) + (0.0 if r is None else np.abs(_np(r)))
    assert (np.abs(_np(out) - ref) <= 1.01 * half * np.abs(ref) + (k + 2) * 2.0 ** -24 * size + 1e-38).all()
    d = _np(dout)
    dy = np.zeros((M, H))
    live = slots >= 0
    dy[slots[live]] = (wn[:, :, None] * d[:, None, :])[live]
    got = _np(leaves[0].grad)
    assert (np.abs(got - dy) <= 1.01 * half * np.abs(dy) + 2.0 ** -24 * np.abs(dy) + 1e-38).all()
    assert (got[kept:] == 0).all()
    if weighted:
        prod = rows * d[:, None, :]
        # sums of H products over 64 lanes and the lanes' six steps
        depth = -(-H // 64) + 8
        assert (np.abs(_np(leaves[1].grad) - prod.sum(2)) <= depth * 2.0 ** -24 * np.abs(prod).sum(2) + 1e-38).all()
    if residual:
        assert torch.equal(leaves[2].grad, dout)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,k,G,H,dropped", [(37, 3, 5, 1024, 0.2), (130, 2, 7, 33, 0.2), (1, 4, 32, 2880, 0.0)])
def test_dispatch_gradient(pkg, dtype, T, k, G, H, dropped):
    plan, gen = _some_plan(pkg, T, k, G, dropped)
    x = torch.randn((T, H), generator=gen).to(dtype).cuda().requires_grad_()
    drows = torch.randn((T * k, H), generator=gen).to(dtype).cuda()
    rows = pkg.dispatch_tokens(x, plan)
    rows.backward(drows)
    terms = _rows_ref(_np(drows), plan.slots.cpu().numpy())
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    ref = terms.sum(1)
    assert (np.abs(_np(x.grad) - ref) <= 1.01 * half * np.abs(ref) + k * 2.0 ** -24 * np.abs(terms).sum(1)).all()


def test_plans_from_elsewhere_stay_inside_the_tensors(pkg):
    """Slots past the rows are skipped, in every direction."""
    offs = torch.tensor([0, 3], device="cuda")
    slots = torch.tensor([[0, 7], [2, -5], [2 ** 31 - 1, 1]], dtype=torch.int32, device="cuda")
    plan = pkg.DispatchPlan(offs, slots)
    x = torch.arange(1, 25, device="cuda", dtype=torch.float32).view(3, 8)
    rows = pkg.dispatch_tokens(x, plan)
    assert torch.equal(rows, torch.stack([x[0], x[2], x[1]] + [torch.zeros_like(x[0])] * 3))
    y = x[:3].clone().requires_grad_()
    out = pkg.combine_tokens(y, plan)
    assert torch.equal(out, torch.stack([y[0], y[2], y[1]]))
    out.sum().backward()
    assert torch.equal(y.grad, torch.ones_like(y))


def test_other_stream_and_graph(pkg):
    """On a stream of its own, and captured: replays on new inputs give what eager calls give."""
    T, E, k, H = 70, 32, 4, 256
    logits, x = torch.empty((T, E), device="cuda"), torch.empty((T, H), dtype=torch.bfloat16, device="cuda")

    def step():
        w, e = pkg.route_experts(logits, k)
        plan = pkg.plan_dispatch(e, E)
        rows = pkg.dispatch_tokens(x, plan)
        return pkg.combine_tokens(rows, plan, w, x), plan.slots, plan.group_offs

    def fill(seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        logits.copy_(torch.randn((T, E), device="cuda", generator=gen))
        x.copy_(torch.randn((T, H), device="cuda", generator=gen))

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(other, step()):
        assert torch.equal(a, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2, 3):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_long_tensors_use_64_bit_offsets(pkg):
    """Rows past 2^32 bytes: 600000 rows of 8192 bf16 are 9.8 GB."""
    T, H = 600000, 8192
    x = torch.zeros((T, H), dtype=torch.bfloat16, device="cuda")
    x[-1] = 3.0
    x[T // 2] = 5.0
    e = torch.zeros((T, 1), dtype=torch.int32, device="cuda")
    e[0] = 1                                             # the first token's row goes last
    plan = pkg.plan_dispatch(e, 2)
    rows = pkg.dispatch_tokens(x, plan)
    assert (rows[T - 2] == 3).all() and (rows[T // 2 - 1] == 5).all() and (rows[T - 1] == 0).all()
    back = pkg.combine_tokens(rows, plan)
    assert torch.equal(back[-1], x[-1]) and torch.equal(back[T // 2], x[T // 2]) and not back[:T // 2].any()


@pytest.mark.parametrize("T,k,G,H,dropped", SIZES)
@pytest.mark.parametrize("which", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)])
def test_combine_gradients_one_by_one(pkg, T, k, G, H, dropped, which):
    """Each gradient by itself is what it is among the others, bit for bit."""
    plan, gen = _some_plan(pkg, T, k, G, dropped)
    parts = [torch.randn((T * k, H), generator=gen), torch.randn((T, k), generator=gen), torch.randn((T, H), generator=gen)]
    dout = torch.randn((T, H), generator=gen).cuda()

    def grads(on):
        leaves = [t.cuda().requires_grad_(bool(g)) for t, g in zip(parts, on)]
        pkg.combine_tokens(leaves[0], plan, leaves[1], leaves[2]).backward(dout)
        return [t.grad for t in leaves]

    for some, full, g in zip(grads(which), grads((1, 1, 1)), which):
        assert (some is not None) == bool(g) and (not g or torch.equal(some, full))
