"""CPU checks of routing, dispatch and combination: the C ABI's refusals (every call fails before any HIP call), the
torch ops' refusals, and the oracle against autograd and differences."""
import os
import re

import numpy as np
import pytest
import torch

from conftest import ROOT
from oracle import moe_oracle as orm

FAKE = 0x100000


def test_header_symbols_exported(pkg):
    text = open(os.path.join(ROOT, "include", "ggemm_moe.h")).read()
    names = sorted(set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(ggemm_moe_\w+)\s*\(", text, re.M)))
    from ggemm_asm_amd import _lib
    assert names == sorted(_lib.MOE_EXPORTS)
    lib = pkg.load_library()
    assert all(hasattr(lib, n) for n in names)


def _route(lib, **kw):
    a = dict(logits=FAKE, dt=1, T=10, E=32, stride=32, k=4, score=0, bias=None, groups=1, top=1, best=2, renorm=1,
             scale=1.0, w=FAKE, e=FAKE)
    a.update(kw)
    return lib.ggemm_moe_route(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(logits=0), -1), (dict(w=0), -1), (dict(e=0), -1), (dict(dt=2), -8), (dict(score=2), -8), (dict(score=-1), -8),
    (dict(T=-1), -2), (dict(E=0), -2), (dict(E=1025, stride=1025), -2), (dict(k=0), -2), (dict(k=33), -2),
    (dict(E=128, stride=128, k=65), -2), (dict(T=2 ** 31), -2), (dict(T=2 ** 29, k=4), -2), (dict(stride=31), -3),
    (dict(logits=FAKE + 2), -4), (dict(logits=FAKE + 1, dt=0), -4), (dict(bias=FAKE + 2), -4), (dict(w=FAKE + 2), -4),
    (dict(groups=5), -2), (dict(groups=0), -2), (dict(groups=4, top=5), -2), (dict(groups=4, top=0), -2),
    (dict(groups=32, best=2), -2), (dict(best=3), -2),
])
def test_route_validation(pkg, kw, rc):
    assert _route(pkg.load_library(), **kw) == rc


def _route_back(lib, **kw):
    a = dict(dw=FAKE, logits=FAKE, dt=1, T=10, E=32, stride=32, k=4, score=0, renorm=1, scale=1.0, e=FAKE, dl=FAKE)
    a.update(kw)
    return lib.ggemm_moe_route_backward(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [(dict(dw=0), -1), (dict(dl=0), -1), (dict(e=0), -1), (dict(E=1025), -2),
                                   (dict(stride=30), -3), (dict(dl=FAKE + 2), -4), (dict(dt=3), -8)])
def test_route_backward_validation(pkg, kw, rc):
    assert _route_back(pkg.load_library(), **kw) == rc


def _plan(lib, **kw):
    a = dict(e=FAKE, n=100, G=8, offs=FAKE, slots=FAKE, ws=FAKE)
    a.update(kw)
    return lib.ggemm_moe_plan(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [(dict(e=0), -1), (dict(offs=0), -1), (dict(slots=0), -1), (dict(ws=0, n=2049), -1),
                                   (dict(n=-1), -2), (dict(n=2 ** 31), -2), (dict(G=0), -2), (dict(G=2048), -2),
                                   (dict(offs=FAKE + 4), -4), (dict(slots=FAKE + 2), -4)])
def test_plan_validation(pkg, kw, rc):
    assert _plan(pkg.load_library(), **kw) == rc


def test_plan_workspace(pkg):
    f = pkg.load_library().ggemm_moe_plan_workspace
    assert f(-1, 8) == 0 and f(10, 0) == 0 and f(10, 2048) == 0
    for n in (2049, 131072, 131073, 2 ** 31 - 256):
        assert 37 <= f(n, 37) <= 256 * 37
    assert f(0, 37) == f(2048, 37) == 0


def _dispatch(lib, **kw):
    a = dict(x=FAKE, rb=64, xs=64, T=10, k=2, slots=FAKE, offs=FAKE, G=4, rows=FAKE, rs=64, M=20)
    a.update(kw)
    return lib.ggemm_moe_dispatch(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [(dict(x=0), -1), (dict(slots=0), -1), (dict(rows=0), -1), (dict(offs=0), -1),
                                   (dict(rb=0), -2), (dict(rb=2 ** 31), -2), (dict(T=-1), -2), (dict(k=0), -2),
                                   (dict(M=2 ** 31), -2), (dict(G=2048), -2), (dict(xs=63), -3), (dict(rs=63), -3),
                                   (dict(slots=FAKE + 1), -4), (dict(offs=FAKE + 4), -4)])
def test_dispatch_validation(pkg, kw, rc):
    assert _dispatch(pkg.load_library(), **kw) == rc


def _combine(lib, **kw):
    a = dict(y=FAKE, dt=0, ys=64, M=20, slots=FAKE, T=10, k=2, w=FAKE, res=FAKE, ress=64, H=64, out=FAKE, outs=64)
    a.update(kw)
    return lib.ggemm_moe_combine(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [(dict(y=0), -1), (dict(out=0), -1), (dict(slots=0), -1), (dict(dt=2), -8),
                                   (dict(H=0), -2), (dict(k=0), -2), (dict(ys=63), -3), (dict(outs=63), -3),
                                   (dict(ress=63), -3), (dict(y=FAKE + 1), -4), (dict(w=FAKE + 2), -4),
                                   (dict(res=FAKE + 2, dt=1), -4)])
def test_combine_validation(pkg, kw, rc):
    assert _combine(pkg.load_library(), **kw) == rc


def _combine_back(lib, **kw):
    a = dict(dout=FAKE, dt=0, ds=64, y=FAKE, ys=64, M=20, slots=FAKE, T=10, k=2, w=FAKE, offs=FAKE, G=4, H=64, dy=FAKE,
             dys=64, dw=FAKE)
    a.update(kw)
    return lib.ggemm_moe_combine_backward(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [(dict(dout=0), -1), (dict(y=0), -1), (dict(offs=0), -1), (dict(slots=0), -1),
                                   (dict(dt=5), -8), (dict(G=0), -2), (dict(H=-1), -2), (dict(ds=1), -3),
                                   (dict(ys=1), -3), (dict(dys=1), -3), (dict(dw=FAKE + 2), -4), (dict(dy=FAKE + 1), -4)])
def test_combine_backward_validation(pkg, kw, rc):
    assert _combine_back(pkg.load_library(), **kw) == rc


# --------------------------------------------------------------------------- the torch ops' refusals

def test_ops_refuse_cpu_tensors(pkg):
    plan = pkg.DispatchPlan(torch.zeros(3, dtype=torch.int64), torch.zeros((2, 1), dtype=torch.int32))
    for f in (lambda: pkg.route_experts(torch.zeros(2, 8), 2), lambda: pkg.plan_dispatch(plan.slots, 2),
              lambda: pkg.dispatch_tokens(torch.zeros(2, 8), plan), lambda: pkg.combine_tokens(torch.zeros(2, 8), plan)):
        with pytest.raises(ValueError, match="GPU"):
            f()


@pytest.fixture
def anywhere(pkg, monkeypatch):
    """The ops' checks without a GPU; nothing may be launched."""
    from ggemm_asm_amd import _lib, moe
    monkeypatch.setattr(moe, "_on_gpu", lambda *a: None)
    monkeypatch.setattr(_lib, "launch", lambda *a: pytest.fail("launched"))


@pytest.mark.parametrize("kw,exc", [
    (dict(logits=torch.zeros(8)), TypeError), (dict(logits=torch.zeros((2, 8), dtype=torch.float16)), TypeError),
    (dict(logits=torch.zeros((2, 1025))), ValueError), (dict(top_k=0), ValueError), (dict(top_k=9), ValueError),
    (dict(logits=torch.zeros((2, 128)), top_k=65), ValueError), (dict(score="relu"), ValueError),
    (dict(num_groups=3), ValueError), (dict(num_groups=4, top_groups=5), ValueError),
    (dict(num_groups=4, top_groups=0), ValueError), (dict(num_groups=8), ValueError), (dict(group_best=3), ValueError),
    (dict(bias=torch.zeros(7)), ValueError), (dict(bias=torch.zeros(8, dtype=torch.bfloat16)), ValueError),
    (dict(bias=torch.zeros(8, device="meta")), ValueError),
])
def test_route_refusals(pkg, anywhere, kw, exc):
    a = dict(logits=torch.zeros((2, 8)), top_k=2)
    a.update(kw)
    with pytest.raises(exc):
        pkg.route_experts(a.pop("logits"), a.pop("top_k"), **a)


def test_exchange_refusals(pkg, anywhere):
    slots, offs = torch.zeros((3, 2), dtype=torch.int32), torch.zeros(5, dtype=torch.int64)
    plan, x = pkg.DispatchPlan(offs, slots), torch.zeros((3, 8))
    y = torch.zeros((6, 8))
    for exc, f in [
            (TypeError, lambda: pkg.plan_dispatch(slots.long(), 4)), (TypeError, lambda: pkg.plan_dispatch(slots[0], 4)),
            (ValueError, lambda: pkg.plan_dispatch(slots, 0)), (ValueError, lambda: pkg.plan_dispatch(slots, 2048)),
            (ValueError, lambda: pkg.dispatch_tokens(x[:2], plan)), (ValueError, lambda: pkg.dispatch_tokens(x[0], plan)),
            (ValueError, lambda: pkg.dispatch_tokens(x, plan, row_align=2)),
            (ValueError, lambda: pkg.dispatch_tokens(x, pkg.DispatchPlan(offs.int(), slots))),
            (ValueError, lambda: pkg.dispatch_tokens(x, pkg.DispatchPlan(offs, slots.long()))),
            (ValueError, lambda: pkg.dispatch_tokens(x, pkg.DispatchPlan(offs.to("meta"), slots))),
            (TypeError, lambda: pkg.combine_tokens(y.half(), plan)),
            (ValueError, lambda: pkg.combine_tokens(y, plan, torch.ones(2, 3))),
            (ValueError, lambda: pkg.combine_tokens(y, plan, torch.ones((3, 2), dtype=torch.bfloat16))),
            (ValueError, lambda: pkg.combine_tokens(y, plan, None, x.bfloat16())),
            (ValueError, lambda: pkg.combine_tokens(y, plan, None, x[:, :4]))]:
        with pytest.raises(exc):
            f()


# --------------------------------------------------------------------------- the oracle

@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
def test_oracle_gradient_is_that_of_its_weights(score, renorm):
    """The oracle's dlogits against central differences of its weights with the experts held."""
    rng = np.random.default_rng(3)
    x, d = rng.normal(size=(5, 12)), rng.normal(size=(5, 3))
    _, e, _ = orm.route(x, 3, score, renormalize=renorm, scale=2.5)
    got = orm.route_backward(d, x, e, score, renorm, 2.5)
    h = 1e-5
    for i in range(12):
        up, dn = x.copy(), x.copy()
        up[:, i] += h
        dn[:, i] -= h
        diff = ((orm.weights_of(up, e, score, renorm, 2.5) - orm.weights_of(dn, e, score, renorm, 2.5)) * d).sum(1) / (2 * h)
        np.testing.assert_allclose(got[:, i], diff, atol=1e-8)


def test_oracle_order():
    x = np.array([[1.0, np.nan, 3.0, 3.0, -np.inf, -0.0, 0.0, np.inf]])
    assert orm.route(x, 8)[1].tolist() == [[1, 7, 2, 3, 0, 5, 6, -1]]
    w, e, _ = orm.route(np.full((1, 4), -np.inf), 2)
    assert e.tolist() == [[-1, -1]] and w.tolist() == [[0.0, 0.0]]
    offs, slots = orm.plan(np.array([[1, 0], [1, -1], [0, 5]]), 3)
    assert offs.tolist() == [0, 2, 4, 4] and slots.tolist() == [[2, 0], [3, -1], [1, -1]]
