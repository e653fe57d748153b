"""The MoE layer on batches whose routing drops tokens (padding: all logits -inf), whatever those tokens hold, and on
views of x."""
import pytest
import torch

pytestmark = pytest.mark.gpu

GATE = dict(slope=1.702, limit=7.0, shift=1.0)


def _layer(pkg, T, E, H, I, seed):
    gen = torch.Generator().manual_seed(seed)

    def make(*s, std=1.0):
        return (torch.randn(s, generator=gen) * std).to(torch.bfloat16).cuda()

    x, logits = make(T, H), make(T, E)
    w = (make(E, 2 * I, H, std=0.1), make(E, H, I, std=0.1))
    biases = dict(bias_up=make(E, 2 * I, std=0.1), bias_down=make(E, H, std=0.1))
    return x, logits, w, lambda x, logits, k: pkg.moe_layer_fp8(x, logits, *w, k, **biases, **GATE)


@pytest.mark.parametrize("T,k,dead", [(1, 2, []), (1, 2, [0]), (3, 1, [1]), (77, 3, [0, 5, 64, 76]), (300, 8, list(range(0, 300, 2))),
                                      (5000, 2, [4999])])
@pytest.mark.parametrize("filler", [3e38, float("inf"), float("-inf"), float("nan")])
def test_masked_tokens_do_not_reach_the_others(pkg, T, k, dead, filler):
    """Without gradients as with them: a dropped token's output is zero and the others' are what they are with zeros in
    its place, bit for bit."""
    x, logits, w, layer = _layer(pkg, T, 8, 128, 96, T + k)
    clean, masked = x.clone(), x.clone()
    logits[dead] = float("-inf")
    clean[dead], masked[dead] = 0.0, filler
    with torch.no_grad():
        want = layer(clean, logits, k)
        got = layer(masked, logits, k)
    assert torch.equal(got, want) and not got[dead].any() and torch.isfinite(got).all()
    assert len(dead) == T or got.any()
    leaf = masked.requires_grad_()
    assert torch.equal(layer(leaf, logits, k), got)


def test_rows_counted_by_their_slots(pkg):
    """The quantizer's amax over the rows that have a slot: one live slot among many, slots outside the rows, both types
    and row lengths on both sides of a wave's step; the rows that do not count are quantized by the same scale."""
    gen = torch.Generator().manual_seed(2)
    for dtype in (torch.bfloat16, torch.float32):
        for T, cols, k in ((1, 8, 1), (5, 512, 64), (130, 2880, 4), (7, 4104, 3), (3000, 72, 2)):
            x = torch.randn((T, cols), generator=gen).to(dtype)
            slots = torch.full((T, k), -1, dtype=torch.int32)
            live = torch.rand(T, generator=gen) < 0.5
            live[T // 2] = True
            at = torch.randint(0, k, (T,), generator=gen)
            slots[torch.arange(T), at] = torch.where(live, torch.arange(T), torch.where(torch.arange(T) % 2 == 0, T * k, -7)).int()
            x[~live] *= 1e4
            q, scale, am = pkg.quantize_fp8_tensorwise(x.cuda(), "e4m3", row_align=128, slots=slots.cuda())
            want = x[live].abs().max().float()
            assert am.item() == want.item()
            full, fscale, _ = pkg.quantize_fp8_tensorwise(x[live].contiguous().cuda(), "e4m3")
            assert torch.equal(scale, fscale)
            assert torch.equal(q[live.cuda()].contiguous().view(torch.uint8), full.view(torch.uint8))
            assert torch.isfinite(q.float()).all()
    none = torch.full((4, 2), -1, dtype=torch.int32, device="cuda")
    q, scale, am = pkg.quantize_fp8_tensorwise(torch.full((4, 16), float("nan"), device="cuda"), slots=none)
    assert am.item() == 0 and scale.item() == 1
    q, scale, am = pkg.quantize_fp8_tensorwise(torch.zeros((0, 16), device="cuda"), slots=none[:0])
    assert tuple(q.shape) == (0, 16) and am.item() == 0 and scale.item() == 1


@pytest.mark.parametrize("view", ["columns", "odd rows", "transposed", "every second", "expanded"])
def test_views_of_x(pkg, view):
    """Rows that start off 16 bytes, rows that lie apart by odd strides, columns that are not contiguous, one row for
    all tokens: both paths take what a copy of x gives."""
    x, logits, w, layer = _layer(pkg, 40, 8, 128, 96, 3)
    wide = torch.zeros((80, 141), dtype=torch.bfloat16, device="cuda")
    if view == "columns":
        wide[:40, 5:133] = x
        v = wide[:40, 5:133]
    elif view == "odd rows":
        wide[:40, :128] = x
        v = wide[:40, :128]
    elif view == "transposed":
        v = x.t().contiguous().t()
    elif view == "every second":
        wide[::2, :128] = x
        v = wide[::2, :128]
    else:
        x = x[:1].expand(40, 128).contiguous()
        v = x[:1].expand(40, 128)
    assert torch.equal(v, x)
    with torch.no_grad():
        want = layer(x, logits, 3)
        assert torch.equal(layer(v, logits, 3), want)
    assert torch.equal(layer(v.detach().requires_grad_(), logits, 3), want)
