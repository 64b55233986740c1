"""Norms around a model's blocks: before one, and where its output joins the residual stream.

    h, stats = norm.forward(x, norm.Norm(w), save=True)                     # before a block
    r, h, s = norm.join(x, y, post=norm.Norm(w1), gate=g, pre=norm.Norm(w2), save=True)
    dx, dy, dgate, dw1, db1, dw2, db2 = norm.join_backward(dr, dh, r, y, *s, post=norm.Norm(w1), gate=g, pre=norm.Norm(w2))

N(v) = (v - m) s weight + bias over the features of a token, with s = 1 / sqrt(mean((v - m)^2) + eps) and m = 0 ("rms") or the
mean ("layer").  A join is r = residual_scale x + scale gate N_post(y), in one pass with the next block's norm h = N_pre(r),
which takes r before it is rounded.  Tensors are tokens x features in BF16 or F16, up to 16384 features, rows any distance
apart; sums are FP32.  Calls follow linear's rules: torch's current stream or `stream`, outputs allocated from it, ChplError.

Autograd does not see these functions; ``normalized`` and ``joined`` are what it differentiates through.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .ckpt8 import on
from ._once import once
from .linear import _choice

_ops = _lib.torch_ops()
KINDS = {"rms": _lib.CHPL_NORM_RMS, "layer": _lib.CHPL_NORM_LAYER}


class Norm(NamedTuple):
    """A norm: weight and bias (or None) of the tensors' type, "rms" or "layer", what is added to the mean square."""
    weight: torch.Tensor
    bias: torch.Tensor | None = None
    kind: str = "rms"
    eps: float = 1e-6


_NONE = (0, None, None, 0.0)


def _of(where: str, v: Norm | None):
    if v is None:
        return _NONE
    weight, bias, kind, eps = v
    code = KINDS.get(kind)
    return _choice(where, "norm", KINDS, kind) if code is None else code, weight, bias, eps


def _gradients(where: str, d: torch.Tensor, dtype, given) -> bool:
    """Whether the parameters' gradients are FP32."""
    if dtype is None and not any(v is not None for v in given):
        return False
    gt = dtype or next((v.dtype for v in given if v is not None), d.dtype)
    if gt is not d.dtype and gt is not torch.float32:
        raise _lib.ChplError(_lib.CHPL_ERR_INVALID, where, f"gradients in {gt}: {d.dtype} or float32 is wanted")
    return gt is torch.float32


def forward(x: torch.Tensor, norm: Norm, *, save: bool = False, out: torch.Tensor | None = None, stream=None):
    """h = N(x); with save=True (h, statistics), what backward wants: tokens x 2, m and s in FP32.  out may be x."""
    if stream is not None:
        with on(stream, x.device):
            return forward(x, norm, save=save, out=out)
    _, h, _, stats = _ops.norm_forward(False, x, None, None, 1.0, 1.0, *_NONE, *_of("norm.forward", norm), save, None, out)
    return (h, stats) if save else h


def backward(dh: torch.Tensor, x: torch.Tensor, stats: torch.Tensor, norm: Norm, *, add: torch.Tensor | None = None,
             need_dx: bool = True, need_dparams: bool = True, dx: torch.Tensor | None = None, dweight: torch.Tensor | None = None,
             dbias: torch.Tensor | None = None, grad_dtype: torch.dtype | None = None, accumulate: bool = False, work=None, stream=None):
    """(dx, dweight, dbias) of h = N(x) from dh; dbias is None where there is no bias.  add is added to dx (the gradient that a
    skip connection brings); dx may be add or dh.  dweight and dbias are of grad_dtype: dh's type, or torch.float32;
    accumulate adds them to the ones given.  work: a uint8 CUDA tensor to use as workspace instead of allocating one; what
    serves a batch serves every smaller one."""
    if stream is not None:
        with on(stream, dh.device):
            return backward(dh, x, stats, norm, add=add, need_dx=need_dx, need_dparams=need_dparams, dx=dx, dweight=dweight, dbias=dbias,
                            grad_dtype=grad_dtype, accumulate=accumulate, work=work)
    f32 = _gradients("norm.backward", dh, grad_dtype, (dweight, dbias))
    out = _ops.norm_backward(False, add, dh, x, None, None, 1.0, 1.0, *_NONE, *_of("norm.backward", norm), None, stats, f32, accumulate,
                             need_dx, False, False, need_dparams, dx, None, None, None, None, dweight, dbias, work)
    return out[0], out[5], out[6]


def join(x: torch.Tensor, y: torch.Tensor, *, post: Norm | None = None, gate: torch.Tensor | None = None, scale: float = 1.0,
         residual_scale: float = 1.0, pre: Norm | None = None, save: bool = False, out: torch.Tensor | None = None,
         out_h: torch.Tensor | None = None, stream=None):
    """r = residual_scale x + scale gate N_post(y); with pre (r, h), h = N_pre(r).  gate: a vector of features, or tokens x
    features.  save=True adds (post statistics, pre statistics), what join_backward wants (None where there is no such norm).
    out may be x or y, out_h may be y."""
    if stream is not None:
        with on(stream, x.device):
            return join(x, y, post=post, gate=gate, scale=scale, residual_scale=residual_scale, pre=pre, save=save, out=out, out_h=out_h)
    r, h, *stats = _ops.norm_forward(True, x, y, gate, scale, residual_scale, *_of("norm.join", post), *_of("norm.join", pre), save, out, out_h)
    got = (r,) if pre is None else (r, h)
    if save:
        return *got, tuple(stats)
    return r if pre is None else got


class Joined(NamedTuple):
    """Gradients of a join; None where there is no such input or it was not asked for."""
    dx: torch.Tensor | None
    dy: torch.Tensor | None
    dgate: torch.Tensor | None
    dpost_weight: torch.Tensor | None
    dpost_bias: torch.Tensor | None
    dpre_weight: torch.Tensor | None
    dpre_bias: torch.Tensor | None


_NOWHERE = Joined(*(None,) * 7)


def join_backward(dr: torch.Tensor | None, dh: torch.Tensor | None, r: torch.Tensor | None, y: torch.Tensor | None,
                  post_stats: torch.Tensor | None, pre_stats: torch.Tensor | None, *, post: Norm | None = None,
                  gate: torch.Tensor | None = None, scale: float = 1.0, residual_scale: float = 1.0, pre: Norm | None = None,
                  need_dx: bool = True, need_dy: bool = True, need_dgate: bool = True, need_dparams: bool = True,
                  into: Joined | None = None, grad_dtype: torch.dtype | None = None, accumulate: bool = False, work=None, stream=None) -> Joined:
    """Gradients of a join from those of r (None: nothing but h uses it) and of h (None where there is no pre).  r is wanted
    with pre, y with post or where the gate's gradient is.  into gives the memory for any of them; its dx may be dr or dh.  A
    vector gate's and the norms' parameters' gradients are of grad_dtype: the tensors' type, or torch.float32; accumulate adds
    them to the ones given.  need_*=False leaves outputs out (None).  work: as backward's."""
    d = dh if dh is not None else dr
    if d is None:
        raise _lib.ChplError(_lib.CHPL_ERR_INVALID, "norm.join_backward", "neither dr nor dh")
    if stream is not None:
        with on(stream, d.device):
            return join_backward(dr, dh, r, y, post_stats, pre_stats, post=post, gate=gate, scale=scale, residual_scale=residual_scale,
                                 pre=pre, need_dx=need_dx, need_dy=need_dy, need_dgate=need_dgate, need_dparams=need_dparams, into=into,
                                 grad_dtype=grad_dtype, accumulate=accumulate, work=work)
    into = into or _NOWHERE
    f32 = False
    if grad_dtype is not None or into is not _NOWHERE:
        f32 = _gradients("norm.join_backward", d, grad_dtype, into[3:] if gate is None or gate.dim() > 1 else into[2:])
    return Joined._make(_ops.norm_backward(True, dr, dh, r, y, gate, scale, residual_scale, *_of("norm.join_backward", post),
                                      *_of("norm.join_backward", pre), post_stats, pre_stats, f32, accumulate, need_dx, need_dy, need_dgate,
                                      need_dparams, *into, work))


# ------------------------------------------------------------------------------------------------------- autograd
def _wanted(*tensors) -> bool:
    return torch.is_grad_enabled() and any(isinstance(v, torch.Tensor) and v.requires_grad for v in tensors)


def _rows(x: torch.Tensor) -> torch.Tensor:
    return x.flatten(0, -2) if x.dim() > 2 else x[None]


class _Normalized(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, kind, eps):
        h, stats = forward(x, Norm(weight, bias, kind, eps), save=True)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.how = kind, eps
        return h

    @staticmethod
    def backward(ctx, dh):
        x, weight, bias, stats = ctx.saved_tensors
        nx, nw, nb = ctx.needs_input_grad[:3]
        with torch.no_grad():
            dx, dw, db = backward(dh.contiguous(), x, stats, Norm(weight, bias, *ctx.how), need_dx=nx, need_dparams=nw or nb)
        return *once("norm.normalized", (dx, dw if nw else None, db if nb else None)), None, None


def normalized(x: torch.Tensor, norm: Norm) -> torch.Tensor:
    """forward(x, norm) as a function that torch's autograd differentiates through, once (a second differentiation raises).
    x has any leading dimensions, features last."""
    if x.dim() not in (0, 2):
        return normalized(_rows(x), norm).reshape(x.shape)
    if _wanted(x, norm.weight, norm.bias):
        return _Normalized.apply(x, *norm)
    return forward(x, norm)


class _Joined(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, post_weight, post_bias, pre_weight, pre_bias, kinds, scales):
        post = None if post_weight is None else Norm(post_weight, post_bias, *kinds[0])
        pre = None if pre_weight is None else Norm(pre_weight, pre_bias, *kinds[1])
        *out, (post_stats, pre_stats) = join(x, y, post=post, gate=gate, scale=scales[0], residual_scale=scales[1], pre=pre, save=True)
        keep_y = post is not None or ctx.needs_input_grad[2]  # a frozen gate's gradients do without it
        ctx.save_for_backward(out[0] if pre else None, y if keep_y else None, gate, post_weight, post_bias, pre_weight, pre_bias,
                              post_stats, pre_stats)
        ctx.how = kinds, scales
        ctx.set_materialize_grads(False)
        return tuple(out) if pre else out[0]

    @staticmethod
    def backward(ctx, dr, dh=None):
        r, y, gate, post_weight, post_bias, pre_weight, pre_bias, post_stats, pre_stats = ctx.saved_tensors
        if dr is None and dh is None:
            return (None,) * 9
        kinds, scales = ctx.how
        post = None if post_weight is None else Norm(post_weight, post_bias, *kinds[0])
        pre = None if dh is None else Norm(pre_weight, pre_bias, *kinds[1])  # an h that nothing uses brings no gradient
        nx, ny, ngate, *nparams = ctx.needs_input_grad[:7]
        with torch.no_grad():
            g = join_backward(None if dr is None else dr.contiguous(), None if dh is None else dh.contiguous(), r, y, post_stats, pre_stats,
                              post=post, gate=gate, scale=scales[0], residual_scale=scales[1], pre=pre, need_dx=nx, need_dy=ny,
                              need_dgate=ngate, need_dparams=any(nparams))
        return *once("norm.joined", g[:3] + tuple(v if n else None for v, n in zip(g[3:], nparams))), None, None


def joined(x: torch.Tensor, y: torch.Tensor, *, post: Norm | None = None, gate: torch.Tensor | None = None, scale: float = 1.0,
           residual_scale: float = 1.0, pre: Norm | None = None):
    """join(x, y, ...) as a function that torch's autograd differentiates through, once.  x and y have any leading dimensions,
    features last; gate is a vector of features or has x's shape."""
    if x.dim() not in (0, 2):
        matrix = gate is not None and gate.dim() > 1
        if y.shape != x.shape or (matrix and gate.shape != x.shape):
            raise _lib.ChplError(_lib.CHPL_ERR_INVALID, "norm.joined", f"x is {tuple(x.shape)}, y {tuple(y.shape)}"
                                 + (f", gate {tuple(gate.shape)}" if matrix else ""))
        out = joined(_rows(x), _rows(y), post=post, gate=_rows(gate) if matrix else gate, scale=scale, residual_scale=residual_scale, pre=pre)
        return out.reshape(x.shape) if pre is None else tuple(v.reshape(x.shape) for v in out)
    params = (*(post or (None, None))[:2], *(pre or (None, None))[:2])
    if _wanted(x, y, gate, *params):
        kinds = tuple(None if v is None else (v.kind, v.eps) for v in (post, pre))
        return _Joined.apply(x, y, gate, *params, kinds, (scale, residual_scale))
    return join(x, y, post=post, gate=gate, scale=scale, residual_scale=residual_scale, pre=pre)
