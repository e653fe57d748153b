"""64-bit reference of expert routing and of the rows' way to the experts and back (numpy, test infrastructure)."""
from __future__ import annotations

import numpy as np


def _order(key):
    """Indices by descending key, NaN first, equal keys by the lower index."""
    nan = np.isnan(key)
    return np.lexsort((np.broadcast_to(np.arange(key.shape[-1]), key.shape), -np.where(nan, 0.0, key), ~nan), axis=-1)


def scores(x, score):
    with np.errstate(all="ignore"):
        if score == "sigmoid":
            return 1.0 / (1.0 + np.exp(-x))
        m = np.nanmax(np.where(np.isnan(x), -np.inf, x), axis=1, keepdims=True)
        e = np.exp(x - np.where(np.isneginf(m), 0.0, m))
        return e / e.sum(1, keepdims=True)


def route(logits, top_k, score="softmax", bias=None, num_groups=1, top_groups=1, group_best=2, renormalize=True,
          scale=1.0):
    """(weights float64 [T, k], experts [T, k], margin [T]): margin is the smallest difference between two unequal
    values that the choice or its order rests on."""
    x = np.asarray(logits, np.float64)
    T, E = x.shape
    p = scores(x, score)
    with np.errstate(all="ignore"):
        key = x.copy() if bias is None and num_groups == 1 else p if bias is None else p + np.asarray(bias, np.float64)
        key = np.where(np.isneginf(x), -np.inf, key)
        margin = np.full(T, np.inf)

        def narrow(a, b):
            d = np.abs(a - b)
            np.minimum(margin, np.where(np.isfinite(d) & (d > 0), d, np.inf), out=margin)

        if num_groups > 1:
            g = key.reshape(T, num_groups, -1)
            best = np.take_along_axis(g, _order(g), 2)[:, :, :group_best].sum(2)
            o = _order(best)
            if top_groups < num_groups:
                v = np.take_along_axis(best, o, 1)
                narrow(v[:, top_groups - 1], v[:, top_groups])
            keep = np.zeros((T, num_groups), bool)
            np.put_along_axis(keep, o[:, :top_groups], True, 1)
            key = np.where(keep[:, :, None], g, -np.inf).reshape(T, E)
        o = _order(key)
        v = np.take_along_axis(key, o, 1)
        for j in range(min(top_k, E - 1)):
            narrow(v[:, j], v[:, j + 1])
        idx = o[:, :top_k]
        live = ~np.isneginf(v[:, :top_k])
        ps = np.where(live, np.take_along_axis(p, idx, 1), 0.0)
        if renormalize and score == "softmax":
            ps = scores(np.where(live, np.take_along_axis(x, idx, 1), -np.inf), "softmax")
        elif renormalize:
            ps = ps / np.maximum(ps.sum(1, keepdims=True), 1e-20)
    return np.where(live, ps, 0.0) * scale, np.where(live, idx, -1), margin


def weights_of(logits, experts, score, renormalize, scale):
    """The weights of given experts (none -1), in 64 bits."""
    x = np.asarray(logits, np.float64)
    if renormalize and score == "softmax":
        return scores(np.take_along_axis(x, experts, 1), "softmax") * scale
    ps = np.take_along_axis(scores(x, score), experts, 1)
    return (ps / np.maximum(ps.sum(1, keepdims=True), 1e-20) if renormalize else ps) * scale


def route_backward(dweights, logits, experts, score, renormalize, scale):
    """dlogits [T, E] of the weights' gradient, in 64 bits."""
    x, d = np.asarray(logits, np.float64), np.asarray(dweights, np.float64) * scale
    out = np.zeros_like(x)
    for t in range(x.shape[0]):
        live = experts[t] >= 0
        e = experts[t][live]
        if e.size == 0:
            continue
        p = scores(x[t:t + 1], score)[0]
        dp = np.zeros(x.shape[1])
        if renormalize and score == "softmax":
            q = scores(x[t:t + 1, e], "softmax")[0]
            out[t, e] = q * (d[t][live] - (d[t][live] * q).sum())
            continue
        if renormalize:
            s = p[e].sum()
            dp[e] = d[t][live] / s - (d[t][live] * p[e]).sum() / s ** 2 if s >= 1e-20 else d[t][live] / 1e-20
        else:
            dp[e] = d[t][live]
        out[t] = p * (1 - p) * dp if score == "sigmoid" else p * (dp - (dp * p).sum())
    return np.where(np.isneginf(x), 0.0, out)


def plan(experts, G):
    """(group_offs [G + 1], slots like experts): rows by expert, then in the order of the choices."""
    flat = np.asarray(experts).ravel()
    slots = np.full(flat.size, -1, np.int64)
    offs = [0]
    for g in range(G):
        at = np.flatnonzero(flat == g)
        slots[at] = offs[-1] + np.arange(at.size)
        offs.append(offs[-1] + at.size)
    return np.array(offs), slots.reshape(np.shape(experts))
