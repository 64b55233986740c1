"""Norms, joins and 4-bit products where calls meet and sizes end: rows past 2^32 bytes, very many tokens, two streams at once,
inference mode, gradients that autograd hands over expanded, functions that carry no graph."""
import pytest
import torch

import linear_ref as lin
import mx4_ref
import norm_ref as ref
from chpl_b200 import check_device, ffn, mx4, norm

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def mk(g, *s, dt=BF, scale=1.0, mean=0.0):
    return torch.empty(*s, device="cuda").normal_(mean, scale, generator=g).to(dt)


def far(v, ld):
    """v's rows, ld apart."""
    full = torch.empty((v.shape[0] - 1) * ld + v.shape[1], dtype=v.dtype, device="cuda")
    out = full.as_strided(v.shape, (ld, 1))
    out.copy_(v)
    return out


@pytest.mark.parametrize("ld", [(1 << 31) + 8, (1 << 31) + 1])
def test_rows_past_32_bits(cuda, ld):
    """Rows 4.3 GB apart, aligned and not: bit for bit the results of rows that lie close together."""
    g = gen(1)
    T, n = 3, 520
    x, y, dh = mk(g, T, n), mk(g, T, n), mk(g, T, n)
    v = norm.Norm(mk(g, n, mean=1.0, scale=0.1), mk(g, n), "layer")
    want = norm.join(x, y, post=v, pre=v, save=True)
    X, O = far(x, ld), far(torch.zeros_like(x), ld)
    got = norm.join(X, y, post=v, pre=v, save=True, out=O)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    w1, w2 = norm.join_backward(y, dh, want[0], y, *want[2], post=v, pre=v), norm.join_backward(y, dh, O, y, *want[2], post=v, pre=v, into=norm.Joined(X, *(None,) * 6))
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(w1, w2))
    del X, O
    X = far(x, ld)
    w = mx4.pack(mk(g, 200, n))
    want, c = mx4.linear(x, w), mx4.pack(x)
    got = mx4.pack(X)
    assert torch.equal(got.codes, c.codes) and torch.equal(mx4.linear(X, w), want)
    back = far(torch.zeros_like(x), ld)
    assert torch.equal(mx4.unpack(c, out=back), mx4.unpack(c))
    del X, back
    if ld % 2 == 0:
        codes = far(c.codes, (1 << 31) + 16)
        assert torch.equal(mx4.linear(mx4.Mx4(codes, c.scales, n, BF), w), want)
    check_device()


@pytest.mark.parametrize("T,n", [(70001, 72), (200003, 8), (20000, 520)])
def test_many_tokens(cuda, T, n):
    g = gen(2)
    x, dh = mk(g, T, n), mk(g, T, n)
    v = norm.Norm(mk(g, n, mean=1.0, scale=0.1), mk(g, n), "layer", 1e-5)
    w = ref.wide(v)
    h, st = norm.forward(x, v, save=True)
    want = ref.apply(x.double(), w)
    lin.check(h, want[0], BF, ref.ERROR * want[1], "h")
    dx, dw, db = norm.backward(dh, x, st, v, grad_dtype=torch.float32)
    (rx, sx), (rw, sw), (rb, sb) = ref.pull(dh.double(), x.double(), st, w)
    lin.check(dx, rx, BF, ref.ERROR * sx, "dx")
    # a thread adds up T / 148 tokens at most, the groups and units some 200 more
    factor = (T / 148 + 256) * 2.0 ** -24 + ref.ERROR
    assert bool(((dw.double() - rw).abs() <= factor * sw).all()) and bool(((db.double() - rb).abs() <= factor * sb).all())
    c = mx4.pack(x)
    code, scales = mx4_ref.pack(x)
    got, s, _, _ = mx4_ref.unpacked(c)
    assert torch.equal(got, code) and torch.equal(s, scales)


def test_two_streams_at_once(cuda):
    """The same operators side by side on two streams, with clusters and with products of different plans."""
    g = gen(3)
    jobs = []
    for T, n in ((300, 9216), (400, 12288), (200, 1030)):
        x, y = mk(g, T, n), mk(g, T, n)
        v = norm.Norm(mk(g, n, mean=1.0, scale=0.1))
        w = mx4.pack(mk(g, 520, n))

        def job(x=x, y=y, v=v, w=w):
            r, h, st = norm.join(x, y, post=v, pre=v, save=True)
            grads = norm.join_backward(y, x, r, y, *st, post=v, pre=v)
            return [r, h, *[t for t in grads if t is not None], mx4.linear(h, w), mx4.linear(h[:3], w)]

        jobs.append((job, job()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for turn in range(6):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                job, want = jobs[(turn + i) % len(jobs)]
                results.append((job(), want))
    torch.cuda.synchronize()
    for got, want in results:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    check_device()


def test_no_graph_inference_mode_and_expanded_gradients(cuda):
    g = gen(4)
    x, w, w1, w2 = mk(g, 2, 40, 64), mk(g, 64, mean=1.0, scale=0.1), mk(g, 128, 64, scale=0.1), mk(g, 64, 128, scale=0.1)
    v = norm.Norm(w)
    for t in (x, w, w1, w2):
        t.requires_grad_()
    flat = x.flatten(0, 1)
    assert not norm.forward(flat, v).requires_grad and not norm.join(flat, flat, pre=v)[1].requires_grad and not mx4.linear(flat, mx4.pack(w1)).requires_grad
    want = ffn.sublayer(x, v, w1, None, w2, None, post=v, pre=v)
    with torch.inference_mode():
        got = ffn.sublayer(x, v, w1, None, w2, None, post=v, pre=v)
    assert all(torch.equal(a, b) and b.is_inference() for a, b in zip(want, got))
    # sum() hands over one element, expanded
    a = torch.autograd.grad(want[0].sum() + want[1].sum(), (x, w, w1, w2))
    out = ffn.sublayer(x, v, w1, None, w2, None, post=v, pre=v)
    b = torch.autograd.grad(out, (x, w, w1, w2), [torch.ones_like(t) for t in out])
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    # an output that nothing uses
    out = ffn.sublayer(x, v, w1, None, w2, None, pre=v)
    c = torch.autograd.grad(out[1], (x, w1), torch.ones_like(out[1]))
    assert all(bool(torch.isfinite(t).all()) for t in c)
