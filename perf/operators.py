"""Workloads of the linear-layer operators: what is run, what it computes, and what it costs.

Four kinds of pass, each through one public entry point of chpl_b200:

  linear  Y = act(X W^T + b) + R, optionally with the pre-activation Z kept (16 bits, or an 8-bit checkpoint)
  grad    dX, dW, db of such a layer from dY, with its input and pre-activation in 16 bits or as 8-bit checkpoints
  ckpt8   an 8-bit checkpoint written and read back
  ffn     a training step's forward and backward through Y = act(X W1^T + b1) W2^T + b2 + X, holding 8-bit checkpoints

X is tokens x k, W is n x k, Y is tokens x n, all row-major.  An 8-bit checkpoint holds, for each group of 32 consecutive
features of a row, a power-of-two step 2^(s - 133), s = the exponent field of the group's largest magnitude as FP32 (7 at
least), and the codes clamp(rint(x / step), -127, 127); a group with an infinity or a NaN reads back as NaN.

The sizes 1024, 4096, 8192 and 16384 are this repository's block sizes and orders; the others are odd or ragged neighbours.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GROUP = 32


def listed():
    return [
        # one token through the widening layer: weights streamed once, nothing to reuse
        dict(name="decode 1", kind="linear", tokens=1, k=4096, n=16384, type="bf16", act="gelu_tanh", residual=False, save="none", pad=0, empty=0),
        # the smallest call: one token through a square layer, where launch latency counts
        dict(name="decode 1 small", kind="linear", tokens=1, k=1024, n=1024, type="f16", act="relu", residual=False, save="none", pad=0, empty=0),
        # a serving batch through the narrowing layer onto the residual stream
        dict(name="decode 24 residual", kind="linear", tokens=24, k=16384, n=4096, type="f16", act="none", residual=True, save="none", pad=0, empty=0),
        # a short prompt with odd sizes and rows that no 16-byte copy can start on, the pre-activation checkpointed
        dict(name="prompt 333 odd", kind="linear", tokens=333, k=1001, n=2051, type="bf16", act="silu", residual=True, save="z8", pad=2, empty=13),
        # a training or prefill batch through the widening layer
        dict(name="prefill 8192", kind="linear", tokens=8192, k=4096, n=16384, type="bf16", act="gelu", residual=False, save="none", pad=0, empty=0),
        # backward of the narrowing layer: its input is recomputed from the 8-bit checkpoint of the pre-activation
        dict(name="grad 8192 ckpt", kind="grad", tokens=8192, k=16384, n=4096, type="bf16", act="none", in_act="gelu", x="8", z="16", add=False, pad=0, empty=0),
        # backward of a layer with its own activation, everything in 16 bits, a ragged batch with padding tokens
        dict(name="grad 2000 act", kind="grad", tokens=2000, k=4096, n=4096, type="bf16", act="silu", in_act="none", x="16", z="16", add=True, pad=8, empty=100),
        # a small odd-sized layer from 8-bit checkpoints of both input and pre-activation
        dict(name="grad 257 odd", kind="grad", tokens=257, k=1031, n=519, type="f16", act="gelu_tanh", in_act="none", x="8", z="8", add=False, pad=1, empty=0),
        # the checkpoint of a widened batch
        dict(name="ckpt8 8192", kind="ckpt8", tokens=8192, k=16384, type="bf16", pad=0, empty=0),
        # a small FP32 tensor whose rows end inside a group
        dict(name="ckpt8 100 f32", kind="ckpt8", tokens=100, k=1001, type="f32", pad=3, empty=5),
        # a training step of the block
        dict(name="ffn 4096", kind="ffn", tokens=4096, k=4096, n=16384, type="bf16", act="gelu", pad=0, empty=0),
        # the same at a small ragged size
        dict(name="ffn 777", kind="ffn", tokens=777, k=1024, n=4096, type="f16", act="relu", pad=0, empty=40),
    ]


#: multiply-adds of the largest listed case of each kind, and elements of the largest checkpoint
LIMIT = {"linear": 8192 * 4096 * 16384, "grad": 8192 * 4096 * 16384, "ffn": 4096 * 4096 * 16384, "ckpt8": 8192 * 16384}


def draw(rng):
    def size(lo, hi):
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return v if rng.random() < 0.5 else min(hi, max(lo, -(-v // 64) * 64))

    kind = rng.choice(["linear", "linear", "grad", "grad", "ckpt8", "ffn"])
    acts = ["none", "relu", "gelu", "gelu_tanh", "silu"]
    c = dict(kind=kind, tokens=int(round(math.exp(rng.uniform(0.0, math.log(8192))))), k=size(64, 16384), type=rng.choice(["bf16", "f16"]))
    c["pad"] = rng.choice([0, 0, 0, 8, 1])
    if kind != "ckpt8":
        c["n"] = size(64, 16384)
        c["tokens"] = max(1, min(c["tokens"], LIMIT[kind] // (c["k"] * c["n"])))
    else:
        c["type"] = rng.choice(["bf16", "f16", "f32"])
    c["empty"] = rng.choice([0, 0, c["tokens"] // 10])
    if kind == "linear":
        c.update(act=rng.choice(acts), residual=rng.random() < 0.5, save=rng.choice(["none", "none", "z", "z8"]))
    elif kind == "grad":
        # an activation is taken once: behind the layer (act) or, with the layer's input recomputed from it, before (in_act)
        act, before = rng.choice(acts), rng.random() < 0.35
        c.update(act="none" if before else act, in_act=act if before else "none", x=rng.choice(["16", "8"]), z=rng.choice(["16", "8"]), add=rng.random() < 0.5)
    elif kind == "ffn":
        c.update(act=rng.choice(acts[1:]))
    return c


# ------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, T, k, pad = TYPES[case["type"]], case["tokens"], case["k"], case["pad"]

    def rows(width, scale=1.0, outliers=False):
        """tokens x width, rows `width + pad` apart, the last `empty` rows (padding tokens) zero."""
        full = torch.empty(T, width + pad, dtype=dt, device="cuda").normal_(0.0, scale, generator=g)
        if outliers:  # a few features run an order of magnitude above the rest, as activations do
            full[:, 5::97] *= 8
        if case["empty"]:
            full[T - case["empty"]:] = 0
        return full[:, :width]

    def weights(n, k):
        return torch.empty(n, k, dtype=dt, device="cuda").normal_(0.0, k ** -0.5, generator=g)

    def vector(n):
        return torch.empty(n, dtype=dt, device="cuda").normal_(0.0, 0.5, generator=g)

    s = {"case": case, "dtype": dt}
    if case["kind"] == "ckpt8":
        s["x"] = rows(k, outliers=True)
        return s
    n = case["n"]
    if case["kind"] == "linear":
        s.update(x=rows(k, outliers=True), w=weights(n, k), b=vector(n), r=rows(n) if case["residual"] else None)
    elif case["kind"] == "grad":
        s.update(dy=rows(n, 0.05), w=weights(n, k), x=rows(k, outliers=True), z=rows(n) if case["act"] != "none" else None,
                 add=rows(k, 0.05) if case["add"] else None)
        if case["x"] == "8":
            s["x"] = quantised(s["x"])
        if case["z"] == "8" and s["z"] is not None:
            s["z"] = quantised(s["z"])
    else:
        s.update(x=rows(k, outliers=True), w1=weights(n, k), b1=vector(n), w2=weights(k, n), b2=vector(k), dy=rows(k, 0.05))
    return s


# -------------------------------------------------------------------------------------------------------- plain forms
def activate(z, act):
    if act == "none":
        return z
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    return z / (1 + torch.exp(-z))  # silu


def slope(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if act == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def quantised(x):
    """(codes, scales) of an 8-bit checkpoint of x: int8 tokens x k, uint8 tokens x ceil(k / 32)."""
    x = x.float()
    T, k = x.shape
    groups = -(-k // GROUP)
    p = torch.zeros(T, groups * GROUP, dtype=torch.float32, device=x.device)
    p[:, :k] = x
    p = p.reshape(T, groups, GROUP)
    e = torch.bitwise_right_shift(p.abs().amax(2).view(torch.int32), 23)  # exponent field of the largest magnitude
    s = e.clamp(7, 254)
    inv = torch.bitwise_left_shift(260 - s, 23).view(torch.float32)       # 2^(133 - s)
    codes = torch.round(p * inv[:, :, None]).clamp(-127, 127)
    bad = e == 255
    codes = torch.where(bad[:, :, None], torch.zeros_like(codes), codes)
    s = torch.where(bad, torch.full_like(s, 255), s)
    return codes.reshape(T, -1)[:, :k].to(torch.int8).contiguous(), s.to(torch.uint8)


def values(c):
    """What a checkpoint (codes, scales) stands for, in FP32; a plain tensor stands for itself."""
    if not isinstance(c, tuple):
        return c.float()
    codes, scales = c
    s = scales.to(torch.int32)
    step = torch.bitwise_left_shift(s - 6, 23).view(torch.float32)        # 2^(s - 133)
    step = torch.where(s == 255, torch.full_like(step, math.nan), step)
    return codes.float() * step.repeat_interleave(GROUP, dim=1)[:, : codes.shape[1]]


def run(s):
    if own:
        return run_own(s)
    c, dt = s["case"], s["dtype"]
    if c["kind"] == "ckpt8":
        return values(quantised(s["x"])).to(dt)
    if c["kind"] == "linear":
        z = s["x"].float() @ s["w"].float().t() + s["b"].float()
        y = activate(z, c["act"])
        y = (y + s["r"].float() if s["r"] is not None else y).to(dt)
        if c["save"] == "none":
            return y
        return y, z.to(dt) if c["save"] == "z" else values(quantised(z)).to(dt)
    if c["kind"] == "grad":
        g = s["dy"].float()
        if c["act"] != "none":
            g = g * slope(values(s["z"]), c["act"])
        x = values(s["x"])
        dx = g @ s["w"].float()
        if c["in_act"] != "none":
            dx = dx * slope(x, c["in_act"])
            x = activate(x, c["in_act"])
        if s["add"] is not None:
            dx = dx + s["add"].float()
        return dx.to(dt), (g.t() @ x).to(dt), g.sum(0).to(dt)
    # ffn
    x, w1, w2, dy = s["x"].float(), s["w1"].float(), s["w2"].float(), s["dy"].float()
    z = x @ w1.t() + s["b1"].float()
    y = activate(z, c["act"]) @ w2.t() + s["b2"].float() + x
    x8, z8 = values(quantised(x)), values(quantised(z))
    dz = (dy @ w2) * slope(z8, c["act"])
    dw2 = dy.t() @ activate(z8, c["act"])
    out = {"y": y, "dx": dz @ w1 + dy, "dw1": dz.t() @ x8, "db1": dz.sum(0), "dw2": dw2, "db2": dy.sum(0)}
    return {name: v.to(dt) for name, v in out.items()}


# --------------------------------------------------------------------------------------------- the framework's own calls
def run_own(s):
    from chpl_b200 import ckpt8, ffn, linear

    c, dt = s["case"], s["dtype"]

    def checkpoint(v):
        return ckpt8.Ckpt8(v[0], v[1], dt) if isinstance(v, tuple) else v

    if c["kind"] == "ckpt8":
        return ckpt8.unpack(ckpt8.pack(s["x"]))
    if c["kind"] == "linear":
        if c["save"] == "none":
            return linear.forward(s["x"], s["w"], s["b"], residual=s["r"], act=c["act"])
        y, z = linear.forward(s["x"], s["w"], s["b"], residual=s["r"], act=c["act"], save=c["save"])
        return y, z if c["save"] == "z" else ckpt8.unpack(z)
    if c["kind"] == "grad":
        return linear.backward(s["dy"], checkpoint(s["x"]), s["w"], act=c["act"], z=checkpoint(s["z"]), in_act=c["in_act"], add=s["add"])
    y, saved = ffn.forward(s["x"], s["w1"], s["b1"], s["w2"], s["b2"], act=c["act"], residual=True, save=True)
    dx, dw1, db1, dw2, db2 = ffn.backward(s["dy"], saved, s["w1"], s["w2"])
    return {"y": y, "dx": dx, "dw1": dw1, "db1": db1, "dw2": dw2, "db2": db2}


# ----------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    funcs = {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu,
             "gelu": torch.nn.functional.gelu, "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}

    def step(biased):
        return torch.ldexp(torch.ones_like(biased, dtype=torch.float64), biased.to(torch.int32) - 133)

    def spread(v, k):
        return v.repeat_interleave(GROUP, dim=1)[:, :k]

    def read(c):
        return c[0].double() * spread(step(c[1]), c[0].shape[1]) if isinstance(c, tuple) else c.double()

    def through(v):
        """The values after an 8-bit checkpoint."""
        k = v.shape[1]
        p = torch.nn.functional.pad(v, (0, -k % GROUP)).reshape(v.shape[0], -1, GROUP)
        top = p.abs().amax(2)
        biased = torch.where(top > 0, torch.frexp(top)[1] + 126, torch.zeros_like(top, dtype=torch.int32)).clamp(min=7)
        st = spread(step(biased), k)
        return torch.clamp(torch.round(v / st), -127, 127) * st

    def slope_of(v, act):
        v = v.detach().requires_grad_(True)
        return torch.autograd.grad(funcs[act](v).sum(), v)[0]

    kind = case["kind"]
    if kind == "ckpt8":
        return through(s["x"].double())
    if kind == "linear":
        z = torch.addmm(s["b"].double(), s["x"].double(), s["w"].double().t())
        y = funcs[case["act"]](z)
        y = y + s["r"].double() if s["r"] is not None else y
        return y if case["save"] == "none" else (y, z if case["save"] == "z" else through(z))
    if kind == "grad":
        g = s["dy"].double()
        g = g * slope_of(read(s["z"]), case["act"]) if case["act"] != "none" else g
        x = read(s["x"])
        dx = torch.mm(g, s["w"].double()) * slope_of(x, case["in_act"])
        dx = dx + s["add"].double() if s["add"] is not None else dx
        return dx, torch.mm(g.t(), funcs[case["in_act"]](x)), torch.einsum("tn->n", g)
    x, w1, w2, dy = (s[name].double() for name in ("x", "w1", "w2", "dy"))
    z = torch.addmm(s["b1"].double(), x, w1.t())
    y = torch.addmm(s["b2"].double(), funcs[case["act"]](z), w2.t()) + x
    z8 = through(z)
    dz = torch.mm(dy, w2) * slope_of(z8, case["act"])
    return {"y": y, "dx": torch.mm(dz, w1) + dy, "dw1": torch.mm(dz.t(), through(x)), "db1": torch.einsum("tn->n", dz),
            "dw2": torch.mm(dy.t(), funcs[case["act"]](z8)), "db2": torch.einsum("tn->n", dy)}


# --------------------------------------------------------------------------------------------------------------- costs
def work(case):
    T, k, e = case["tokens"], case["k"], 4 if case["type"] == "f32" else 2

    def ckpt(width):
        return T * (width + -(-width // GROUP))

    if case["kind"] == "ckpt8":  # read and coded, then the codes read and the values written
        return {"bytes": 2 * e * T * k + 2 * ckpt(k), "flops": 4 * T * k}
    n = case["n"]
    if case["kind"] == "linear":
        b = e * (T * k + n * k + n + T * n) + (e * T * n if case["residual"] else 0)
        b += {"none": 0, "z": e * T * n, "z8": ckpt(n)}[case["save"]]
        return {"bytes": b, "flops": 2 * T * n * k}
    if case["kind"] == "grad":
        b = e * (T * n + n * k + T * k + n * k + n)                       # dY, W, dX, dW, db
        b += ckpt(k) if case["x"] == "8" else e * T * k
        b += (ckpt(n) if case["z"] == "8" else e * T * n) if case["act"] != "none" else 0
        b += e * T * k if case["add"] else 0
        return {"bytes": b, "flops": 4 * T * n * k}
    # ffn: x, w1, b1, w2, b2, dy in; y, dx and the four gradients out; the checkpoints of x and z written and read once
    return {"bytes": e * (4 * T * k + 4 * n * k + 2 * (n + k)) + 2 * (ckpt(k) + ckpt(n)), "flops": 12 * T * n * k}
