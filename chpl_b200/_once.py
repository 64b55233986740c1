"""Gradients that cannot be differentiated again.  torch's once_differentiable raises only where the incoming gradient carries
a graph; the gradients of these operators depend on their weights and inputs too."""
from __future__ import annotations

import torch

from . import _lib


class _Once(torch.autograd.Function):
    @staticmethod
    def forward(ctx, where, *grads):
        ctx.where = where
        return tuple(v if v is None else v.view_as(v) for v in grads)

    @staticmethod
    def backward(ctx, *_):
        raise _lib.ChplError(_lib.CHPL_ERR_UNSUPPORTED, ctx.where, "its gradients cannot be differentiated again")


def once(where: str, grads):
    """What an operator's backward returns; under create_graph, such that a second differentiation raises."""
    if not torch.is_grad_enabled():
        return tuple(grads)
    return _Once.apply(where, *(v if v is None else v.requires_grad_() for v in grads))
