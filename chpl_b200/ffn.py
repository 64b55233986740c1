"""A model's feed-forward block, Y = act(X W1^T + b1) W2^T + b2 [+ X], trained from 8-bit checkpoints.

Between the passes the block holds X and the pre-activation Z in 8 bits (2.06 bytes per token for each pair of an input
and a hidden feature, where X, Z and act(Z) in 16 bits hold 6): the forward products code Z in their epilogue, and the
backward ones take act(Z), act'(Z) and X from the codes.  The gradients are those of the block at the checkpointed X and Z.

    y, saved = ffn.forward(x, w1, b1, w2, b2, act="gelu", residual=True, save=True)
    dx, dw1, db1, dw2, db2 = ffn.backward(dy, saved, w1, w2)

``block`` wraps the two for torch's autograd; the two themselves it does not see.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib, ckpt8, linear


class Saved(NamedTuple):
    x: ckpt8.Ckpt8
    z: ckpt8.Ckpt8
    act: str
    residual: bool


def forward(x, w1, b1, w2, b2, *, act: str = "gelu", residual: bool = False, save: bool = False, stream=None):
    """Y, or with save=True (Y, what backward needs).  b1 and b2 may be None."""
    if not save:
        h = linear.forward(x, w1, b1, act=act, stream=stream)
        return linear.forward(h, w2, b2, residual=x if residual else None, stream=stream)
    x8 = ckpt8.pack(x, stream=stream)
    h, z8 = linear.forward(x, w1, b1, act=act, save="z8", stream=stream)
    y = linear.forward(h, w2, b2, residual=x if residual else None, stream=stream)
    return y, Saved(x8, z8, act, residual)


def backward(dy, saved: Saved, w1, w2, *, need_dx: bool = True, need_dw1: bool = True, need_dw2: bool = True,
             need_db: bool = True, grad_dtype=None, stream=None):
    """(dx, dw1, db1, dw2, db2) of the block from dy.  need_*=False leaves an output out (None), and the products that
    only it needs; need_db stands for both biases."""
    inner = need_dx or need_dw1 or need_db  # dZ is wanted
    dz, dw2, db2, *db1 = linear.backward(dy, saved.z, w2, in_act=saved.act, need_dx=inner, need_dw=need_dw2, need_db=need_db,
                                         dx_sum=need_db, grad_dtype=grad_dtype, stream=stream)
    dx = dw1 = None
    if need_dx or need_dw1:
        dx, dw1, _ = linear.backward(dz, saved.x, w1, add=dy if saved.residual else None, need_dx=need_dx, need_dw=need_dw1,
                                     need_db=False, grad_dtype=grad_dtype, stream=stream)
    return dx, dw1, db1[0] if db1 else None, dw2, db2


class _Once(torch.autograd.Function):
    """Gradients that cannot be differentiated again.  torch's once_differentiable raises only where dy carries a graph;
    the block's gradients depend on its weights and input too."""

    @staticmethod
    def forward(ctx, *grads):
        return tuple(v if v is None else v.view_as(v) for v in grads)

    @staticmethod
    def backward(ctx, *_):
        raise _lib.ChplError(_lib.CHPL_ERR_UNSUPPORTED, "ffn.block", "its gradients cannot be differentiated again")


class _Block(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, act, residual):
        y, s = forward(x, w1, b1, w2, b2, act=act, residual=residual, save=True)
        ctx.save_for_backward(s.x.codes, s.x.scales, s.z.codes, s.z.scales, w1, w2)
        ctx.how = (x.dtype, act, residual)
        return y

    @staticmethod
    def backward(ctx, dy):
        xc, xs, zc, zs, w1, w2 = ctx.saved_tensors
        dt, act, residual = ctx.how
        s = Saved(ckpt8.Ckpt8(xc, xs, dt), ckpt8.Ckpt8(zc, zs, dt), act, residual)
        x, n1, v1, n2, v2 = ctx.needs_input_grad[:5]
        with torch.no_grad():
            dx, dw1, db1, dw2, db2 = backward(dy.contiguous(), s, w1, w2, need_dx=x, need_dw1=n1, need_dw2=n2, need_db=v1 or v2)
        grads = [dx, dw1, db1 if v1 else None, dw2, db2 if v2 else None]
        if torch.is_grad_enabled():  # create_graph
            grads = _Once.apply(*(v if v is None else v.requires_grad_() for v in grads))
        return *grads, None, None


def block(x, w1, b1, w2, b2, act: str = "gelu", residual: bool = False):
    """The block as a function that torch's autograd differentiates through, once: its gradients cannot be differentiated
    again (create_graph and a second backward pass raise).  x has any leading dimensions, rows of features last.  Where
    no gradient can be asked for, nothing is held; a frozen weight's gradient is not formed."""
    if isinstance(x, torch.Tensor) and x.dim() not in (0, 2):
        y = block(x.flatten(0, -2) if x.dim() > 2 else x[None], w1, b1, w2, b2, act, residual)
        return y.reshape(*x.shape[:-1], y.shape[1])
    if torch.is_grad_enabled() and any(isinstance(v, torch.Tensor) and v.requires_grad for v in (x, w1, b1, w2, b2)):
        return _Block.apply(x, w1, b1, w2, b2, act, residual)
    return forward(x, w1, b1, w2, b2, act=act, residual=residual)
