"""Workloads of the operators around and inside a feed-forward block: its norms and residual joins, and 4-bit products.

Six kinds of pass, each through one public entry point of chpl_b200:

  norm       h = N(x): RMS or layer norm of a token's features, before a block
  norm_grad  dx, dweight, dbias of it, the skip connection's gradient added to dx
  join       r = beta x + alpha gate * Npost(y), h = Npre(r): a block's output y normed, gated and scaled onto the residual
             stream x, and the next block's norm of the sum
  join_grad  the gradients of that
  pack       a tensor coded in microscaled 4-bit floating point, and read back
  product    Y = act(Q(X) W^T + b) + R with W in that format and X coded on the way

N(v) = (v - m) s w + b with m the mean (layer) or 0 (rms) and s = 1 / sqrt(mean((v - m)^2) + eps); h in a join is the norm of r
before r is rounded.  The 4-bit format: 32 consecutive features of a row share a step 2^(s - 127), s = max(e, 7) - 2 for the
exponent field e of their largest magnitude as FP32, and each is x / step rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6
and their negatives, ties to the even code, larger ones to 6 (OCP Microscaling MXFP4).

The sizes 1024, 4096, 8192 and 16384 are this repository's block sizes and orders; the others are odd or ragged neighbours.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GROUP = 32
EPS = 1e-6


def listed():
    return [
        # one token before a block while text is generated: latency
        dict(name="norm 1", kind="norm", tokens=1, n=4096, type="bf16", norm="rms", pad=0, empty=0),
        # a prompt of odd width, its rows apart and unaligned
        dict(name="norm 777 odd", kind="norm", tokens=777, n=1001, type="f16", norm="layer", pad=2, empty=13),
        # the norm before a block, trained, with the skip connection's gradient
        dict(name="norm_grad 8192", kind="norm_grad", tokens=8192, n=4096, type="bf16", norm="layer", add=True, pad=0, empty=0),
        # between two blocks: norm after the one, learned gate, residual scale, norm before the next
        dict(name="join 8192", kind="join", tokens=8192, n=4096, type="bf16", post="rms", gate="vector", pre="rms", alpha=0.5, beta=1.0, pad=0, empty=0),
        # a serving batch on a wide stream, every token with a gate of its own
        dict(name="join 24 wide", kind="join", tokens=24, n=16384, type="f16", post="layer", gate="matrix", pre="layer", alpha=1.0, beta=0.75, pad=0, empty=0),
        # the same joins trained
        dict(name="join_grad 8192", kind="join_grad", tokens=8192, n=4096, type="bf16", post="rms", gate="vector", pre="rms", alpha=0.5, beta=1.0, pad=0, empty=0),
        dict(name="join_grad 333 odd", kind="join_grad", tokens=333, n=1031, type="f16", post="layer", gate="matrix", pre="layer", alpha=1.0, beta=0.75, pad=1, empty=20),
        # a layer's weights, or a large batch, coded and read back
        dict(name="pack 8192", kind="pack", tokens=8192, n=16384, type="bf16", pad=0, empty=0),
        # a small FP32 tensor whose rows end inside a group
        dict(name="pack 100 f32", kind="pack", tokens=100, n=1001, type="f32", pad=3, empty=5),
        # one token through the widening layer: weights streamed once
        dict(name="product 1", kind="product", tokens=1, k=4096, n=16384, type="bf16", act="gelu_tanh", residual=False, pad=0, empty=0),
        # a short prompt with odd sizes onto the residual stream
        dict(name="product 333 odd", kind="product", tokens=333, k=1001, n=2051, type="f16", act="silu", residual=True, pad=2, empty=13),
        # a prefill batch through the widening layer
        dict(name="product 8192", kind="product", tokens=8192, k=4096, n=16384, type="bf16", act="gelu", residual=False, pad=0, empty=0),
    ]


#: elements of the largest row-wise case and multiply-adds of the largest product
ELEMENTS = {"norm": 8192 * 8192, "norm_grad": 8192 * 4096, "join": 8192 * 4096, "join_grad": 8192 * 4096, "pack": 8192 * 16384}
PRODUCTS = 8192 * 4096 * 16384


def draw(rng):
    def size(lo, hi):
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return v if rng.random() < 0.5 else min(hi, max(lo, -(-v // 64) * 64))

    kind = rng.choice(["norm", "norm_grad", "join", "join_grad", "pack", "product", "product", "product"])
    c = dict(kind=kind, tokens=int(round(math.exp(rng.uniform(0.0, math.log(8192))))), n=size(64, 16384), type=rng.choice(["bf16", "f16"]))
    if kind == "product":
        c["k"] = size(64, 16384)
        c["tokens"] = max(1, min(c["tokens"], PRODUCTS // (c["k"] * c["n"])))
        c.update(act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), residual=rng.random() < 0.5)
    else:
        c["tokens"] = max(1, min(c["tokens"], ELEMENTS[kind] // c["n"]))
    c["pad"] = rng.choice([0, 0, 0, 8, 1])
    c["empty"] = rng.choice([0, 0, c["tokens"] // 10])
    if kind in ("norm", "norm_grad"):
        c["norm"] = rng.choice(["rms", "layer"])
        if kind == "norm_grad":
            c["add"] = rng.random() < 0.5
    elif kind in ("join", "join_grad"):
        c.update(post=rng.choice(["none", "rms", "layer"]), gate=rng.choice(["none", "vector", "matrix"]), pre=rng.choice(["none", "rms", "layer"]),
                 alpha=rng.choice([1.0, 0.5]), beta=rng.choice([1.0, 0.75]))
    elif kind == "pack":
        c["type"] = rng.choice(["bf16", "f16", "f32"])
    return c


# ------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, T, pad, kind = TYPES[case["type"]], case["tokens"], case["pad"], case["kind"]

    def rows(width, scale=1.0, outliers=False):
        """tokens x width, rows `width + pad` apart, the last `empty` rows (padding tokens) zero."""
        full = torch.empty(T, width + pad, dtype=dt, device="cuda").normal_(0.0, scale, generator=g)
        if outliers:  # a few features run an order of magnitude above the rest, as activations do
            full[:, 5::97] *= 8
        if case["empty"]:
            full[T - case["empty"]:] = 0
        return full[:, :width]

    def vector(n, mean=0.0, scale=0.3):
        return torch.empty(n, dtype=dt, device="cuda").normal_(mean, scale, generator=g)

    def norm(how, n):
        """(weight, bias, kind) of a norm; a layer norm has a bias."""
        if how == "none":
            return None
        return vector(n, 1.0), vector(n) if how == "layer" else None, how

    n = case["n"]
    s = {"case": case, "dtype": dt}
    if kind == "norm":
        s.update(x=rows(n, outliers=True), norm=norm(case["norm"], n))
    elif kind == "norm_grad":
        s.update(x=rows(n, outliers=True), norm=norm(case["norm"], n), dh=rows(n, 0.05), add=rows(n, 0.05) if case["add"] else None)
        s["stats"] = statistics(s["x"].float(), case["norm"])
    elif kind in ("join", "join_grad"):
        s.update(x=rows(n, outliers=True), y=rows(n), post=norm(case["post"], n), pre=norm(case["pre"], n),
                 gate={"none": lambda: None, "vector": lambda: vector(n), "matrix": lambda: rows(n, 0.5)}[case["gate"]]())
        if kind == "join_grad":  # what the forward pass kept
            r = joined(s)
            s.update(r=rows(n), dr=rows(n, 0.05), dh=rows(n, 0.05) if s["pre"] else None)
            s["r"].copy_(r.to(dt))
            s["post_stats"] = statistics(s["y"].float(), case["post"]) if s["post"] else None
            s["pre_stats"] = statistics(r, case["pre"]) if s["pre"] else None
            del s["x"]
    elif kind == "pack":
        s["x"] = rows(n, outliers=True)
    else:
        k = case["k"]
        w = torch.empty(n, k, dtype=dt, device="cuda").normal_(0.0, k ** -0.5, generator=g)
        s.update(x=rows(k, outliers=True), b=vector(n), r=rows(n) if case["residual"] else None)
        if own:
            from chpl_b200 import mx4
            s["w"] = mx4.pack(w)
        else:
            s["w"] = quantised(w)
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


def statistics(v, how):
    """(mean, 1 / deviation) of every row: tokens x 2, FP32."""
    mean = v.mean(1) if how == "layer" else torch.zeros_like(v[:, 0])
    return torch.stack([mean, 1 / torch.sqrt((v - mean[:, None]).square().mean(1) + EPS)], dim=1)


def normed(v, norm):
    st = statistics(v, norm[2])
    h = (v - st[:, :1]) * st[:, 1:] * norm[0].float()
    return h + norm[1].float() if norm[1] is not None else h


def norm_gradients(d, v, st, norm):
    """(dv, dweight, dbias) of normed(v, norm) from its gradient d, all FP32."""
    g, hat = d * norm[0].float(), (v - st[:, :1]) * st[:, 1:]
    inner = g - hat * (g * hat).mean(1, keepdim=True)
    if norm[2] == "layer":
        inner = inner - g.mean(1, keepdim=True)
    return inner * st[:, 1:], (d * hat).sum(0), d.sum(0) if norm[1] is not None else None


def joined(s):
    p = normed(s["y"].float(), s["post"]) if s["post"] else s["y"].float()
    if s["gate"] is not None:
        p = p * s["gate"].float()
    return s["case"]["beta"] * s["x"].float() + s["case"]["alpha"] * p


LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantised(x):
    """(codes, scales) of x in the 4-bit format: uint8 rows x n (sign * 8 + index of the level), uint8 rows x ceil(n / 32)."""
    x = x.float()
    T, n = x.shape
    groups = -(-n // GROUP)
    p = torch.zeros(T, groups * GROUP, dtype=torch.float32, device=x.device)
    p[:, :n] = x
    p = p.reshape(T, groups, GROUP)
    e = torch.bitwise_right_shift(p.abs().amax(2).view(torch.int32), 23)  # exponent field of the largest magnitude
    s = e.clamp(7, 254) - 2
    inv = torch.bitwise_left_shift(254 - s, 23).view(torch.float32)       # 2^(127 - s)
    q = p * inv[:, :, None]
    a = q.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    for i, (lo, hi) in enumerate(zip(LEVELS, LEVELS[1:])):                # past the midpoint, or on it where the upper code is even
        code += (a > (lo + hi) / 2) if i % 2 == 0 else (a >= (lo + hi) / 2)
    code += 8 * (q < 0)
    bad = e == 255
    code = torch.where(bad[:, :, None], torch.zeros_like(code), code)
    s = torch.where(bad, torch.full_like(s, 255), s)
    return code.reshape(T, -1)[:, :n].contiguous(), s.to(torch.uint8)


def values(c):
    """What codes and scales stand for, in FP32."""
    codes, scales = c
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float32, device=codes.device)
    s = scales.to(torch.int32)
    step = torch.bitwise_left_shift(s, 23).view(torch.float32)            # 2^(s - 127)
    step = torch.where(s == 255, torch.full_like(step, math.nan), step)
    return table[codes.int()] * step.repeat_interleave(GROUP, dim=1)[:, : codes.shape[1]]


def run(s):
    if own:
        return run_own(s)
    c, dt, kind = s["case"], s["dtype"], s["case"]["kind"]

    def rounded(out):
        return {name: v.to(dt) for name, v in out.items() if v is not None}

    if kind == "norm":
        return normed(s["x"].float(), s["norm"]).to(dt)
    if kind == "norm_grad":
        dx, dw, db = norm_gradients(s["dh"].float(), s["x"].float(), s["stats"], s["norm"])
        return rounded({"dx": dx + s["add"].float() if s["add"] is not None else dx, "dw": dw, "db": db})
    if kind == "join":
        r = joined(s)
        return rounded({"r": r, "h": normed(r, s["pre"]) if s["pre"] else None})
    if kind == "join_grad":
        d, dw_pre, db_pre = s["dr"].float(), None, None
        if s["pre"]:
            dv, dw_pre, db_pre = norm_gradients(s["dh"].float(), s["r"].float(), s["pre_stats"], s["pre"])
            d = d + dv
        do = c["alpha"] * d
        y = s["y"].float()
        dp, dgate = do, None
        if s["gate"] is not None:
            p = y
            if s["post"]:
                p = (y - s["post_stats"][:, :1]) * s["post_stats"][:, 1:] * s["post"][0].float()
                p = p + s["post"][1].float() if s["post"][1] is not None else p
            dp = do * s["gate"].float()
            dgate = (do * p).sum(0) if c["gate"] == "vector" else do * p
        dy, dw_post, db_post = norm_gradients(dp, y, s["post_stats"], s["post"]) if s["post"] else (dp, None, None)
        return rounded({"dx": c["beta"] * d, "dy": dy, "dgate": dgate, "dw_post": dw_post, "db_post": db_post, "dw_pre": dw_pre, "db_pre": db_pre})
    if kind == "pack":
        return values(quantised(s["x"])).to(dt)
    y = activate(values(quantised(s["x"])) @ values(s["w"]).t() + s["b"].float(), c["act"])
    return (y + s["r"].float() if s["r"] is not None else y).to(dt)


# --------------------------------------------------------------------------------------------- the framework's own calls
def run_own(s):
    from chpl_b200 import mx4, norm

    c, kind = s["case"], s["case"]["kind"]

    def of(parts):
        return norm.Norm(parts[0], parts[1], kind=parts[2], eps=EPS) if parts else None

    if kind == "norm":
        return norm.forward(s["x"], of(s["norm"]))
    if kind == "norm_grad":
        out = norm.backward(s["dh"], s["x"], s["stats"], of(s["norm"]), add=s["add"])
        return {name: v for name, v in zip(("dx", "dw", "db"), out) if v is not None}
    how = dict(post=of(s.get("post")), gate=s.get("gate"), scale=c.get("alpha", 1.0), residual_scale=c.get("beta", 1.0), pre=of(s.get("pre")))
    if kind == "join":
        out = norm.join(s["x"], s["y"], **how)
        return {"r": out[0], "h": out[1]} if s["pre"] else {"r": out}
    if kind == "join_grad":
        out = norm.join_backward(s["dr"], s["dh"], s["r"], s["y"], s["post_stats"], s["pre_stats"], **how)
        names = ("dx", "dy", "dgate", "dw_post", "db_post", "dw_pre", "db_pre")
        return {name: v for name, v in zip(names, out) if v is not None}
    if kind == "pack":
        return mx4.unpack(mx4.pack(s["x"]))
    return mx4.linear(s["x"], s["w"], s["b"], residual=s["r"], act=c["act"])


# ----------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    kind = case["kind"]

    def wide(v):
        return None if v is None else v.double()

    def coded(v):
        """The values after the 4-bit format."""
        n = v.shape[1]
        p = torch.nn.functional.pad(v, (0, -n % GROUP)).reshape(v.shape[0], -1, GROUP)
        top = p.abs().amax(2, keepdim=True)
        low = torch.full_like(top, 7, dtype=torch.int32)
        biased = torch.where(top > 0, torch.frexp(top)[1] + 126, low).clamp(min=7)
        q = torch.ldexp(p, 129 - biased)
        quantum = torch.ldexp(torch.ones_like(q), torch.frexp(q.abs().clamp(min=1.0))[1] - 2)
        q = torch.clamp(torch.round(q / quantum) * quantum, -6.0, 6.0)
        return torch.ldexp(q, biased - 129).reshape(v.shape[0], -1)[:, :n]

    def read(codes, scales):
        magnitude = (codes & 7).int()
        m = torch.where(magnitude < 2, magnitude.double() / 2, torch.ldexp(1 + (magnitude & 1).double() / 2, (magnitude >> 1) - 1))
        sign = 1 - 2 * (codes >> 3).double()
        return torch.ldexp(sign * m, scales.int().repeat_interleave(GROUP, dim=1)[:, : codes.shape[1]] - 127)

    def hat(v, how, st=None):
        if st is not None:
            return (v - st[:, 0:1].double()) * st[:, 1:2].double()
        c = v - torch.einsum("tn->t", v)[:, None] / v.shape[1] if how == "layer" else v
        return c / torch.sqrt(torch.einsum("tn,tn->t", c, c)[:, None] / v.shape[1] + EPS)

    def apply(norm, v, st=None):
        h = torch.einsum("tn,n->tn", hat(v, norm[2], st), norm[0].double())
        return h if norm[1] is None else h + norm[1].double()

    def pull(norm, d, v, st):
        """Gradients of apply by the quotient rule's projection: d weight, without its parts along the hat and the ones."""
        xh = hat(v, norm[2], st)
        g = torch.einsum("tn,n->tn", d, norm[0].double())
        along = torch.einsum("tn,tn->t", g, xh) / v.shape[1]
        mean = torch.einsum("tn->t", g) / v.shape[1] if norm[2] == "layer" else torch.zeros_like(along)
        dv = torch.einsum("tn,t->tn", g - mean[:, None] - torch.einsum("t,tn->tn", along, xh), st[:, 1].double())
        return dv, torch.einsum("tn,tn->n", d, xh), None if norm[1] is None else torch.einsum("tn->n", d)

    def present(**out):
        return {name: v for name, v in out.items() if v is not None}

    if kind == "norm":
        return apply(s["norm"], wide(s["x"]))
    if kind == "norm_grad":
        dx, dw, db = pull(s["norm"], wide(s["dh"]), wide(s["x"]), s["stats"])
        return present(dx=dx if s["add"] is None else dx + wide(s["add"]), dw=dw, db=db)
    if kind == "join":
        p = apply(s["post"], wide(s["y"])) if s["post"] else wide(s["y"])
        r = torch.add(case["beta"] * wide(s["x"]), p if s["gate"] is None else p * wide(s["gate"]), alpha=case["alpha"])
        return present(r=r, h=apply(s["pre"], r) if s["pre"] else None)
    if kind == "join_grad":
        pre = pull(s["pre"], wide(s["dh"]), wide(s["r"]), s["pre_stats"]) if s["pre"] else (0.0, None, None)
        d, y, gate = wide(s["dr"]) + pre[0], wide(s["y"]), wide(s["gate"])
        dp = case["alpha"] * (d if gate is None else d * gate)
        post = pull(s["post"], dp, y, s["post_stats"]) if s["post"] else (dp, None, None)
        dgate = None
        if gate is not None:
            p = apply(s["post"], y, s["post_stats"]) if s["post"] else y
            dgate = case["alpha"] * (torch.einsum("tn,tn->n", d, p) if case["gate"] == "vector" else d * p)
        return present(dx=case["beta"] * d, dy=post[0], dgate=dgate, dw_post=post[1], db_post=post[2], dw_pre=pre[1], db_pre=pre[2])
    if kind == "pack":
        return coded(wide(s["x"]))
    funcs = {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu,
             "gelu": torch.nn.functional.gelu, "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}
    y = funcs[case["act"]](torch.addmm(wide(s["b"]), coded(wide(s["x"])), read(*s["w"]).t()))
    return y if s["r"] is None else y + wide(s["r"])


# --------------------------------------------------------------------------------------------------------------- costs
def work(case):
    T, n, e, kind = case["tokens"], case["n"], 4 if case["type"] == "f32" else 2, case["kind"]

    def coded(width):
        return -(-width // 2) + -(-width // GROUP)

    def vectors(how):
        return {"none": 0, "rms": 1, "layer": 2}[how]

    if kind == "norm":
        return {"bytes": e * (2 * T * n + vectors(case["norm"]) * n), "flops": 6 * T * n}
    if kind == "norm_grad":  # dh, x, statistics, add, weight in; dx, dweight, dbias out
        return {"bytes": e * ((3 + case["add"]) * T * n + (1 + vectors(case["norm"])) * n) + 8 * T, "flops": 14 * T * n}
    if kind in ("join", "join_grad"):
        gate = {"none": 0, "vector": n, "matrix": T * n}[case["gate"]]
        pre, post = case["pre"] != "none", case["post"] != "none"
        if kind == "join":  # x, y, gate in; r, h out
            return {"bytes": e * ((3 + pre) * T * n + gate + (vectors(case["post"]) + vectors(case["pre"])) * n), "flops": (4 + 6 * pre + 6 * post) * T * n}
        # dr, gate in; dx, dy, dgate out; y where a norm or a gate wants it, dh and r where there is a next norm
        needs_y = post or case["gate"] != "none"
        weights = (vectors(case["post"]) + post + vectors(case["pre"]) + pre) * n
        return {"bytes": e * ((3 + needs_y + 2 * pre) * T * n + 2 * gate + weights) + 8 * T * (pre + post), "flops": (4 + 12 * pre + 14 * post) * T * n}
    if kind == "pack":  # read and coded, then the codes read and the values written
        return {"bytes": 2 * T * (e * n + coded(n)), "flops": 4 * T * n}
    k = case["k"]
    return {"bytes": e * (T * k + n + T * n * (2 if case["residual"] else 1)) + n * coded(k), "flops": 2 * T * n * k}
