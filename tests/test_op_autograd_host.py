"""CPU checks of what autograd sees of the ops: which tensors get gradients, what is kept for them, and that
derivatives the ops do not have are refused. Launches are replaced by nothing: values are arbitrary here."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

E4, BF = torch.float8_e4m3fn, torch.bfloat16


@pytest.fixture
def unlaunched(pkg, monkeypatch):
    from ggemm_asm_amd import _lib, moe, product
    calls = []
    monkeypatch.setattr(_lib, "launch", lambda name, dev, sizes, *args: calls.append((name, args)))
    for m in (moe, product):
        monkeypatch.setattr(m, "_on_gpu", lambda *a: None)
    return calls


def _plan(pkg, T=4, k=2, G=3):
    return pkg.DispatchPlan(torch.zeros(G + 1, dtype=torch.int64), torch.zeros((T, k), dtype=torch.int32))


# name: (inputs that may require a gradient, the call on them)
def _ops(pkg):
    plan = _plan(pkg)
    y, w, res = torch.randn(8, 16), torch.randn(4, 2), torch.randn(4, 16)
    return {
        "route": ([torch.randn(4, 6)], lambda x: pkg.route_experts(x, 2)[0]),
        "dispatch": ([torch.randn(4, 16)], lambda x: pkg.dispatch_tokens(x, plan)),
        "combine": ([y, w, res], lambda a, b, c: pkg.combine_tokens(a, plan, b, c)),
        "product": ([torch.randn(3, 64), torch.randn((8, 32)).to(BF)], lambda b, r: _product(pkg, b, r, "swiglu")),
    }


def _product(pkg, bias, residual, activation, **kw):
    a, b = torch.zeros((8, 32), dtype=E4), torch.zeros((3, 64, 32), dtype=E4)
    return pkg.grouped_gemm_fp8_bias_act(a, b, torch.ones(()), torch.ones(()), torch.tensor([0, 2, 2, 6]), bias, activation,
                                         residual, **kw)


# --------------------------------------------------------------------------- bias and residual of the product

@pytest.mark.parametrize("activation", [None, "silu", "swiglu"])
@pytest.mark.parametrize("which", ["bias", "residual", "both"])
@pytest.mark.parametrize("keep", [False, True])
def test_product_keeps_the_graph_of_bias_and_residual(pkg, unlaunched, activation, which, keep):
    bias = torch.randn((3, 64), dtype=BF).requires_grad_(which != "residual")
    residual = torch.randn((8, 32 if activation == "swiglu" else 64)).to(BF).requires_grad_(which != "bias")
    got = _product(pkg, bias, residual, activation, keep_preact=keep)
    out = got[0] if keep else got
    assert out.requires_grad and (not keep or not got[1].requires_grad)
    assert [n for n, _ in unlaunched] == ["ggemm_product_fp8_bias_act"]
    with torch.no_grad():
        out.copy_(torch.zeros_like(out))
    dout = torch.randn(out.shape).to(BF)
    out.backward(dout)
    if which != "residual":
        assert bias.grad.dtype == BF and tuple(bias.grad.shape) == (3, 64)
    else:
        assert bias.grad is None
    if which != "bias":
        want = dout.clone()
        want[6:] = 0                                  # rows of no group: the result does not depend on the residual there
        assert torch.equal(residual.grad, want)
    else:
        assert residual.grad is None
    assert [n for n, _ in unlaunched[1:]] == ([] if which == "residual" else ["ggemm_product_act_backward"])


def test_product_without_gradients_keeps_nothing(pkg, unlaunched):
    bias = torch.randn((3, 64)).requires_grad_()
    with torch.no_grad():
        assert not _product(pkg, bias, None, "silu").requires_grad
    assert not _product(pkg, bias.detach(), None, "silu").requires_grad
    assert all(args[3] is None for _, args in unlaunched)          # no z is written


# --------------------------------------------------------------------------- derivatives that there are not

@pytest.mark.parametrize("op", ["route", "dispatch", "combine", "product"])
def test_second_derivatives_are_refused(pkg, unlaunched, op):
    inputs, f = _ops(pkg)[op]
    inputs = [t.requires_grad_() for t in inputs]
    out = f(*inputs)
    d = torch.randn_like(out).requires_grad_()
    grads = torch.autograd.grad(out, inputs, d, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        sum(g.float().sum() for g in grads).backward()


def test_every_backward_is_once_differentiable(pkg):
    from ggemm_asm_amd import autograd, moe, product
    for m in (autograd, moe, product):
        for f in vars(m).values():
            if isinstance(f, type) and issubclass(f, torch.autograd.Function) and f is not torch.autograd.Function:
                assert hasattr(f.backward, "__wrapped__"), f


@pytest.mark.parametrize("op", ["route", "dispatch", "combine", "product"])
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(pkg, unlaunched, op, grad):
    """Forward-mode derivatives of each input, with reverse mode on or off: an error, not a result without them."""
    inputs, f = _ops(pkg)[op]
    for i in range(len(inputs)):
        with fwAD.dual_level(), torch.set_grad_enabled(grad):
            args = [fwAD.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(inputs)]
            with pytest.raises(RuntimeError, match="jvp"):
                f(*args)
            assert not f(*inputs).requires_grad


# --------------------------------------------------------------------------- what is kept

def test_combine_keeps_only_what_its_gradients_read(pkg, unlaunched):
    """y for the weights' gradient, the weights for y's."""
    plan = _plan(pkg)
    for grads, kept in (((1, 0, 0), "w"), ((0, 1, 0), "y"), ((1, 1, 0), "yw"), ((0, 0, 1), ""), ((1, 0, 1), "w")):
        t = {n: v.requires_grad_(bool(g)) for (n, v), g in
             zip(dict(y=torch.randn(8, 16), w=torch.randn(4, 2), r=torch.randn(4, 16)).items(), grads)}
        out = pkg.combine_tokens(t["y"], plan, t["w"], t["r"])
        held = {s.data_ptr() for s in out.grad_fn.saved_tensors if s is not None}
        assert {n for n in "yw" if t[n].data_ptr() in held} == set(kept), grads
        out.backward(torch.randn_like(out))
        for (n, v), g in zip(t.items(), grads):
            assert (v.grad is not None) == bool(g) and (not g or v.grad.shape == v.shape)


def test_combine_gradient_of_y_alone_reads_no_y(pkg, unlaunched):
    y = torch.randn(8, 16).requires_grad_()
    pkg.combine_tokens(y, _plan(pkg), torch.randn(4, 2)).sum().backward()
    name, args = unlaunched[-1]
    assert name == "ggemm_moe_combine_backward" and args[3] is None and args[-1] is None
