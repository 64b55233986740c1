"""The norm before a block, the block, and its join with the residual stream run together, as a model's layer is trained and
served: ffn.sublayer, and the same through the passes that it is made of."""
import pytest
import torch

import linear_ref as lin
import norm_ref as ref
from chpl_b200 import check_device, ffn, mx4, norm

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def layer(T, d, hidden, dt, seed, kind="rms", matrix=False, lead=()):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def mk(*s, scale=1.0, mean=0.0):
        return torch.empty(*s, device="cuda").normal_(mean, scale, generator=g).to(dt)

    bias = (lambda: mk(d, scale=0.1)) if kind == "layer" else (lambda: None)
    n = [norm.Norm(mk(d, scale=0.1, mean=1.0), bias(), kind, 1e-5) for _ in range(3)]
    return dict(x=mk(*lead, T, d), norm=n[0], w1=mk(hidden, d, scale=d ** -0.5), b1=mk(hidden, scale=0.1), w2=mk(d, hidden, scale=hidden ** -0.5),
                b2=mk(d, scale=0.1), post=n[1], gate=mk(*lead, T, d, scale=0.5) if matrix else mk(d, scale=0.5), scale=0.5, residual_scale=0.75, pre=n[2])


def leaves(p):
    t = [p["x"], p["w1"], p["b1"], p["w2"], p["b2"], p["gate"]]
    for n in (p["norm"], p["post"], p["pre"]):
        t += [v for v in n[:2] if v is not None]
    return t


@pytest.mark.parametrize("T,d,hidden,dt,kind,matrix", [(1, 64, 128, BF, "rms", False), (77, 264, 1000, HF, "layer", True), (600, 512, 2048, BF, "rms", True),
                                                       (300, 1024, 1024, BF, "layer", False)])
def test_training_step_is_its_passes(cuda, T, d, hidden, dt, kind, matrix):
    """Autograd's outputs and gradients are bit for bit those of the passes; x's two gradients are added in their type."""
    p = layer(T, d, hidden, dt, 1, kind, matrix)
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    dr, dn = (torch.empty(T, d, device="cuda").normal_(0.0, 0.1, generator=g).to(dt) for _ in range(2))
    how = {k: p[k] for k in ("post", "gate", "scale", "residual_scale", "pre")}
    h, st = norm.forward(p["x"], p["norm"], save=True)
    y, saved = ffn.forward(h, p["w1"], p["b1"], p["w2"], p["b2"], save=True)
    r, n, stats = norm.join(p["x"], y, save=True, **how)
    j = norm.join_backward(dr, dn, r, y, *stats, **how)
    dh, dw1, db1, dw2, db2 = ffn.backward(j.dy, saved, p["w1"], p["w2"])
    dx, dw, db = norm.backward(dh, p["x"], st, p["norm"])
    want = [j.dx + dx, dw1, db1, dw2, db2, j.dgate, dw, db, j.dpost_weight, j.dpost_bias, j.dpre_weight, j.dpre_bias]
    t = [v.requires_grad_() for v in leaves(p)]
    out = ffn.sublayer(**p)
    assert torch.equal(out[0], r) and torch.equal(out[1], n)
    got = torch.autograd.grad(out, t, (dr, dn))
    want = [v for v in want if v is not None]
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
    check_device()


def test_training_step_against_64_bits(cuda):
    """2-norm errors.  Outputs: h, act(z), y and the result are rounded once each, 4 u, and one more for FP32 sums.  Gradients: X
    and Z come from 8-bit codes with an rms error of a step / sqrt(12), a step being at most 2^-6 of the group's largest, some
    2.5 to 4.5 deviations: up to 0.02 of a deviation, which reaches a gradient once through X and, times |act''| < 1.2, once or
    twice through Z: 0.05 with the roundings."""
    p = layer(300, 512, 1024, BF, 3, "layer", True, lead=(2,))
    t = [v.requires_grad_() for v in leaves(p)]
    out = ffn.sublayer(**p)
    d = [torch.randn_like(v) for v in out]
    got = torch.autograd.grad(out, t, d)
    w = {k: v.detach().double().requires_grad_() if isinstance(v, torch.Tensor) else v for k, v in p.items()}
    for k in ("norm", "post", "pre"):
        w[k] = norm.Norm(p[k].weight.detach().double().requires_grad_(), p[k].bias.detach().double().requires_grad_(), p[k].kind, p[k].eps)

    def N(v, n):
        c = v - v.mean(-1, keepdim=True)
        return c / (c.square().mean(-1, keepdim=True) + n.eps).sqrt() * n.weight + n.bias

    y = lin.act(N(w["x"], w["norm"]) @ w["w1"].t() + w["b1"], "gelu") @ w["w2"].t() + w["b2"]
    r = 0.75 * w["x"] + 0.5 * w["gate"] * N(y, w["post"])
    want = (r, N(r, w["pre"]))
    for a, b in zip(out, want):
        assert (a.double() - b).norm() <= 5 * lin.UNIT[BF] * b.norm()
    for a, b in zip(got, torch.autograd.grad(want, leaves(w), [v.double() for v in d])):
        assert a.shape == b.shape and (a.double() - b).norm() <= 0.05 * b.norm()


@pytest.mark.parametrize("T", [1, 5, 200])
def test_serving_in_4_bits(cuda, T):
    """With coded weights, and nothing to train, the sublayer is its passes bit for bit, one token as a batch's row: the products
    of a row do not depend on its neighbours where they take the same tile."""
    p = layer(T, 512, 1024, BF, 5)
    p["w1"], p["w2"] = mx4.pack(p["w1"]), mx4.pack(p["w2"])
    r, n = ffn.sublayer(**p)
    h = norm.forward(p["x"], p["norm"])
    y = mx4.linear(mx4.linear(h, p["w1"], p["b1"], act="gelu"), p["w2"], p["b2"])
    want = norm.join(p["x"], y, post=p["post"], gate=p["gate"], scale=0.5, residual_scale=0.75, pre=p["pre"])
    assert torch.equal(r, want[0]) and torch.equal(n, want[1])
    check_device()


def test_captured_step(cuda):
    """Forward and backward captured into a graph and replayed on new inputs.  No eager graph of the same leaves may live
    meanwhile: torch keeps a leaf's gradient node, with the stream that it was made on, as long as one does, and a captured
    backward pass of any function then waits for a stream outside of the capture, which torch refuses."""
    p = layer(130, 256, 512, BF, 6)
    t = [v.requires_grad_() for v in leaves(p)]
    dr, dn = (torch.randn(130, 256, device="cuda", dtype=BF) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ffn.sublayer(**p), t, (dr, dn))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ffn.sublayer(**p)
        grads = torch.autograd.grad(out, t, (dr, dn))
    for seed in (1, 2):
        torch.manual_seed(seed)
        with torch.no_grad():
            p["x"].copy_(torch.randn_like(p["x"]))
            dr.copy_(torch.randn_like(dr))
        graph.replay()
        want = ffn.sublayer(**p)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(want, t, (dr, dn))))
    check_device()
