"""The workspace of the norms' gradients: what serves a batch serves every smaller one, wherever its operands lie."""
import ctypes

import pytest
import torch

from chpl_b200 import _lib, norm

P = [4096 * (i + 1) for i in range(32)]  # addresses that are never looked at
LD = ("lddr", "lddh", "ldr", "ldy", "ldgate", "lddx", "lddy", "lddgate")
SUMS = dict(dpost_weight=P[10], dpost_bias=P[11], dpre_weight=P[12], dpre_bias=P[13])


def need(tokens, n, pad=0, at=0, join=1, dgate=P[9], vector=False, **sums):
    v = _lib.Norm(kind=_lib.CHPL_NORM_LAYER, eps=1e-6, weight=P[20] + at, bias=P[21] + at)
    a = _lib.NormBwd(type=0, join=join, grad_type=0, tokens=tokens, n=n, scale=1.0, residual_scale=1.0, dr=P[0] + at, dh=P[1] + at, r=P[2] + at, y=P[3] + at,
                     gate=P[4] + at if join else None, post=v if join else _lib.Norm(), pre=v, post_stats=P[5], pre_stats=P[6], dx=P[7] + at,
                     dy=P[8] + at if join else None, dgate=dgate if join else None, **{**{k: n + pad for k in LD}, **({"ldgate": 0} if vector else {})},
                     **{k: p for k, p in SUMS.items() if sums.get(k, join or k.startswith("dpre"))})
    size = ctypes.c_size_t()
    assert _lib.load().chpl_norm_backward_worksize(ctypes.byref(a), ctypes.byref(size)) == 0
    return size.value


WIDTHS = (1, 64, 500, 512, 513, 1024, 2048, 4096, 5120, 8192, 9000, 12288, 16384)


@pytest.mark.parametrize("join,vector", [(0, False), (1, False), (1, True)])
def test_never_falls(join, vector):
    tokens = (*range(1, 320), 443, 444, 445, 1000, 4096, 100000, 1 << 30)
    before = [0] * len(tokens)
    for n in WIDTHS:
        sizes = [need(t, n, join=join, vector=vector) for t in tokens]
        assert all(a <= b for a, b in zip(sizes, sizes[1:])), n  # in tokens
        assert all(a <= b for a, b in zip(before, sizes)), n     # in n
        before = sizes


@pytest.mark.parametrize("n", WIDTHS)
def test_where_operands_lie_is_the_same(n):
    for tokens in (1, 75, 148, 149, 297, 5000):
        for join in (0, 1):
            assert len({need(tokens, n, pad, at, join) for pad, at in ((0, 0), (8, 0), (1, 0), (0, 2), (3, 2))}) == 1


def test_fewer_outputs_need_no_more():
    for n in (520, 4096, 12288):
        for tokens in (1, 148, 149, 3000):
            all_ = need(tokens, n)
            assert need(tokens, n, dpre_bias=False) <= all_ and need(tokens, n, dpost_weight=False, dpost_bias=False) <= all_
            assert need(tokens, n, dgate=None) <= all_ and need(tokens, n, **{k: False for k in SUMS}) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n,pad", [(4096, 0), (5120, 0), (1031, 1), (12288, 8)])
def test_smaller_batches_run_in_a_larger_ones_workspace(cuda, n, pad):
    """Whatever the batch, in the memory for 149 tokens, bit for bit the results in memory of its own."""
    g = torch.Generator(device="cuda")
    g.manual_seed(n)

    def mk(*s):
        return torch.empty(*s, device="cuda").normal_(generator=g).bfloat16()

    v, gate = norm.Norm(mk(n), mk(n), "layer"), mk(n)
    work = torch.empty(need(149, n, vector=True), dtype=torch.uint8, device="cuda")
    full = [mk(149, n + pad) for _ in range(4)]
    for T in (149, 148, 147, 75, 74, 1):
        x, y, dr, dh = (t[:T, :n] for t in full)
        r, _, st = norm.join(x, y, post=v, gate=gate, pre=v, save=True)
        how = dict(post=v, gate=gate, pre=v)
        want = norm.join_backward(dr, dh, r, y, *st, **how)
        got = norm.join_backward(dr, dh, r, y, *st, **how, work=work)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        want = norm.backward(dh, r, st[1], v)
        got = norm.backward(dh, r, st[1], v, work=work)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
