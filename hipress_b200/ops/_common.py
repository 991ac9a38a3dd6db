"""What the layer operators share: checks of arguments, the CPU forms' numbers, first derivatives."""
from __future__ import annotations

import functools

import torch

TYPES = (torch.float32, torch.bfloat16, torch.float16)


def same_device(what, *ts):
    dev = ts[0].device
    for t in ts[1:]:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: tensors on {dev} and {t.device}")
    return dev


def wide(x):
    return x if x.dtype == torch.float64 else x.float()   # CPU: float64 is taken as it is


class _Refused(torch.autograd.Function):
    """A value as it is, which cannot be differentiated by what it was made from."""

    @staticmethod
    def forward(ctx, x, *made_from):
        return x.view_as(x)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("a gradient of a layer operator cannot be differentiated")


def first_order(backward):
    """For a backward pass whose results have no graph; the node has saved all its inputs.  Where a graph is
    wanted (``create_graph``) the results say so when they are differentiated, whether or not the
    gradient that came in has a graph itself."""
    @functools.wraps(backward)
    def run(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        made_from = [t for t in (*ctx.saved_tensors, *grads) if t is not None and t.requires_grad]
        # what is handed on unchanged keeps the graph that it has
        return tuple(g if g is None or any(g is x for x in grads) else _Refused.apply(g.detach(), *made_from) for g in out)
    return run
