"""Coding into given memory: what is returned is of the type of what was coded, whatever the memory held before."""
import types

import pytest
import torch

from chpl_b200 import ckpt8, linear, mx4

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("held", [BF, HF, FP])
@pytest.mark.parametrize("dt", [BF, HF, FP])
def test_mx4_type(monkeypatch, held, dt):
    monkeypatch.setattr(mx4, "_ops", types.SimpleNamespace(mx4_pack=lambda x, codes, scales: (codes, scales)))
    out = mx4.Mx4(torch.empty(3, 32, dtype=torch.uint8), torch.empty(1024, dtype=torch.uint8), 40, held)
    got = mx4.pack(torch.empty(3, 40, dtype=dt), out=out)
    assert got.dtype is dt and got.codes is out.codes and got.scales is out.scales and got.cols == 40 and (got is out) == (dt is held)


@pytest.mark.parametrize("held", [BF, HF, FP])
@pytest.mark.parametrize("dt", [BF, HF, FP])
def test_ckpt8_type(monkeypatch, held, dt):
    monkeypatch.setattr(ckpt8, "_ops", types.SimpleNamespace(ckpt8_pack=lambda x, codes, scales: (codes, scales)))
    monkeypatch.setattr(linear, "_ops", types.SimpleNamespace(linear_forward=lambda x, *a: (None, *a[7:9])))
    out = ckpt8.empty(3, 40, held, "cpu")
    x = torch.empty(3, 40, dtype=dt)
    for got in (ckpt8.pack(x, out=out), linear.forward(x, None, save="z8", z=out)[1]):
        assert got.dtype is dt and got.codes is out.codes and got.scales is out.scales and (got is out) == (dt is held)


@pytest.mark.gpu
def test_mx4_memory_of_another_type(cuda):
    """A buffer of bfloat16 codes used again for float16 rows: products and values come in float16."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x, w = (torch.empty(5, 96, device="cuda").normal_(generator=g).half() for _ in range(2))
    w4 = mx4.pack(w)
    c = mx4.pack(x, out=mx4.pack(torch.zeros(5, 96, dtype=BF, device="cuda")))
    assert torch.equal(mx4.linear(c, w4), mx4.linear(x, w4)) and mx4.linear(c, w4).dtype is HF
    assert torch.equal(mx4.unpack(c), mx4.unpack(mx4.pack(x))) and mx4.unpack(c).dtype is HF


@pytest.mark.gpu
def test_ckpt8_memory_of_another_type(cuda):
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    x, w = (torch.empty(5, 96, device="cuda").normal_(generator=g).half() for _ in range(2))
    c = ckpt8.pack(x, out=ckpt8.empty(5, 96, BF, "cuda"))
    assert ckpt8.unpack(c).dtype is HF and torch.equal(ckpt8.unpack(c), ckpt8.unpack(ckpt8.pack(x)))
    z = linear.forward(x, w, save="z8", z=ckpt8.empty(5, 5, BF, "cuda"))[1]
    assert ckpt8.unpack(z).dtype is HF and torch.equal(ckpt8.unpack(z), ckpt8.unpack(linear.forward(x, w, save="z8")[1]))
