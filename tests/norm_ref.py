"""Plain FP64 restatements of norms and joins and of their gradients, with the sizes of what is added up in them, from which
the tests' bounds follow.

The kernels' arithmetic is FP32: a value that comes of some k roundings of terms of size s is off by at most k 2^-24 s.  The
longest chains are the sums over a row: sixteen features a thread, 5 + 5 steps through the lanes of a warp and of the row's
warps, and up to 4 CTAs; with the products, the mean, the square root and the weights fewer than 100 roundings in all, so
2^-17 of the terms' sizes bounds them (100 2^-24 < 2^-17).  A sum over T tokens has T and some 60 further terms in a row."""
from typing import NamedTuple

import torch

ERROR = 2.0 ** -17


class N(NamedTuple):
    """A norm in FP64: weight, bias, kind, eps."""
    weight: torch.Tensor
    bias: torch.Tensor | None
    kind: str
    eps: float


def wide(norm):
    return None if norm is None else N(norm.weight.double(), None if norm.bias is None else norm.bias.double(), norm.kind, norm.eps)


def stats(v, norm):
    m = v.mean(1) if norm.kind == "layer" else torch.zeros_like(v[:, 0])
    return torch.stack([m, 1 / torch.sqrt(((v - m[:, None]) ** 2).mean(1) + norm.eps)], 1)


def apply(v, norm):
    """(N(v), size of its terms)."""
    st = stats(v, norm)
    h = (v - st[:, :1]) * st[:, 1:] * norm.weight
    size = (v.abs() + v.abs().mean(1, keepdim=True)) * st[:, 1:] * norm.weight.abs()
    return (h, size) if norm.bias is None else (h + norm.bias, size + norm.bias.abs())


def pull(d, v, st, norm):
    """((dv, size), (dweight, size), (dbias, size)) of N at v from its gradient d; size: of the terms that are added up."""
    st = st.double()
    s, xh = st[:, 1:], (v - st[:, :1]) * st[:, 1:]
    a = (v.abs() + st[:, :1].abs()) * s  # size of xh's terms
    g = d * norm.weight
    inner = g - xh * (g * xh).mean(1, keepdim=True)
    size = g.abs() + a * (g.abs() * a).mean(1, keepdim=True)
    if norm.kind == "layer":
        inner, size = inner - g.mean(1, keepdim=True), size + g.abs().mean(1, keepdim=True)
    db = None if norm.bias is None else (d.sum(0), d.abs().sum(0))
    return (inner * s, size * s), ((d * xh).sum(0), (d.abs() * a).sum(0)), db


def join(x, y, post, gate, scale, residual_scale, pre):
    """{"r": (value, size), "h": ...}"""
    p, ps = apply(y, post) if post else (y, y.abs())
    if gate is not None:
        p, ps = p * gate, ps * gate.abs()
    r = residual_scale * x + scale * p
    rs = abs(residual_scale) * x.abs() + abs(scale) * ps
    out = {"r": (r, rs)}
    if pre:
        # r's error goes into h through its own term and through the row's statistics
        h, hs = apply(r, pre)
        st = stats(r, pre)
        out["h"] = (h, hs + (rs + rs.mean(1, keepdim=True) * (1 + (r.abs() * st[:, 1:]))) * st[:, 1:] * pre.weight.abs())
    return out


def join_backward(dr, dh, r, y, post_stats, pre_stats, post, gate, scale, residual_scale, pre):
    """{name: (value, size)} of what norm.join_backward returns."""
    D = torch.zeros_like(y) if dr is None else dr
    Ds = D.abs()
    out = {}
    if pre:
        (dv, dvs), out["dpre_weight"], out["dpre_bias"] = pull(dh, r, pre_stats, pre)
        D, Ds = D + dv, Ds + dvs
    out["dx"] = (residual_scale * D, abs(residual_scale) * Ds)
    do, dos = scale * D, abs(scale) * Ds
    dp, dps = do, dos
    if gate is not None:
        st = None if post is None else post_stats.double()
        p = y if post is None else (y - st[:, :1]) * st[:, 1:] * post.weight + (0 if post.bias is None else post.bias)
        ps = y.abs() if post is None else (y.abs() + st[:, :1].abs()) * st[:, 1:] * post.weight.abs() + (0 if post.bias is None else post.bias.abs())
        dg, dgs = do * p, dos * ps
        out["dgate"] = (dg, dgs) if gate.dim() == 2 else (dg.sum(0), dgs.sum(0))
        dp, dps = do * gate, dos * gate.abs()
    if post:
        out["dy"], out["dpost_weight"], out["dpost_bias"] = pull(dp, y, post_stats, post)
        # the error of dp goes through the same sums
        g, st = dps * post.weight.abs(), post_stats.double()
        a = (y.abs() + st[:, :1].abs()) * st[:, 1:]
        out["dy"] = (out["dy"][0], (g + g.mean(1, keepdim=True) + a * (g * a).mean(1, keepdim=True)) * st[:, 1:])
        out["dpost_weight"] = (out["dpost_weight"][0], (dps * a).sum(0))
        if post.bias is not None:
            out["dpost_bias"] = (out["dpost_bias"][0], dps.sum(0))
    else:
        out["dy"] = (dp, dps)
    return {name: v for name, v in out.items() if v is not None}


def sum_error(tokens):
    return (tokens + 64) * 2.0 ** -24 + ERROR
