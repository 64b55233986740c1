"""Plain FP64 restatements of the linear-layer operators and of the 8-bit checkpoint, and the error bounds of their tests."""
import math

import torch

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
GROUP = 32
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # unit roundoffs
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}  # half the least subnormal


def act(z, name):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "gelu":
        return z * 0.5 * torch.erfc(-z * math.sqrt(0.5))
    if name == "gelu_tanh":
        return z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * torch.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = 2 * math.sqrt(2 / math.pi)
        s = 1 / (1 + torch.exp(-c * (z + 0.044715 * z ** 3)))
        return s + z * s * (1 - s) * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s + z * s * (1 - s)
    return torch.ones_like(z)


def pack(x):
    """(codes int8, scales uint8) by the rule of include/chpl.h, element by element in FP64."""
    x = x.double()
    rows, cols = x.shape
    groups = -(-cols // GROUP)
    p = torch.zeros(rows, groups * GROUP, dtype=torch.float64, device=x.device)
    p[:, :cols] = x
    p = p.reshape(rows, groups, GROUP)
    bad = ~torch.isfinite(p).all(2)
    top = torch.where(bad, torch.zeros_like(p[:, :, 0]), p.abs().amax(2))
    s = torch.where(top >= 2.0 ** -126, torch.frexp(top)[1] + 126, torch.zeros_like(top, dtype=torch.int32)).clamp(min=7)
    step = torch.ldexp(torch.ones_like(top), s - 133)
    codes = torch.round(torch.nan_to_num(p, 0, 0, 0) / step[:, :, None]).clamp(-127, 127)
    codes = torch.where(bad[:, :, None], torch.zeros_like(codes), codes)
    s = torch.where(bad, torch.full_like(s, 255), s)
    return codes.reshape(rows, -1)[:, :cols].to(torch.int8), s.to(torch.uint8)


def unpack(codes, scales):
    step = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.to(torch.int32) - 133)
    step = torch.where(scales == 255, torch.full_like(step, math.nan), step)
    return codes.double() * step.repeat_interleave(GROUP, dim=1)[:, : codes.shape[1]]


def forward(x, w, b, r, name):
    """(Y, Z, sum |x||w| + |b|) in FP64."""
    z = x.double() @ w.double().t()
    size = x.double().abs() @ w.double().abs().t()
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    y = act(z, name)
    return (y + r.double() if r is not None else y), z, size


# The kernels round each product exactly, add in FP32 (an error of at most 2^-23 of the running magnitude per addition,
# rounded or cut), and evaluate act and act' to 2^-18 of their argument (or of 1); |act'| < 1.2.
def add_error(terms):
    return (terms + 2) * 2.0 ** -23


ACT_ERROR = 2.0 ** -18


def check(got, ref, dtype, slack, what, roundings=1):
    """|got - ref| <= u |ref| + slack elementwise; in the 2-norm, u for each of the `roundings` roundings of operands and
    result (a relative error of at most u each), plus the slack's norm over 8 (accumulation errors do not all have their
    bound's size and one sign) as far as it stays below one more u."""
    u = UNIT[dtype]
    got = got.double()
    assert got.shape == ref.shape
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    fine = torch.isfinite(ref) & torch.isfinite(got)
    d, ref = torch.where(fine, (got - ref).abs(), 0.0), torch.where(fine, ref, 0.0)
    slack = torch.where(fine, slack, 0.0) if isinstance(slack, torch.Tensor) else slack
    bound = u * ref.abs() + slack + TINY[dtype]
    worst = (d - bound).max().item() if d.numel() else -1
    assert worst <= 0, f"{what}: off by {d.max().item()}, {worst} over its bound"
    if d.numel():
        extra = torch.as_tensor(slack, device=d.device, dtype=torch.float64).expand_as(d).norm().item() / 8
        lim = roundings * u * ref.norm().item() + min(extra, u * ref.norm().item()) + TINY[dtype] * d.numel() ** 0.5
        assert d.norm().item() <= lim, f"{what}: 2-norm error {d.norm().item()} over {lim}"
