"""The end of a model: log probabilities of given tokens, and the loss that is their mean.

    p = token_log_probs(logits, tokens, top=5)      p.log_probs, p.entropy, p.top_log_probs, p.top_tokens
    loss = cross_entropy(logits, labels)

CUDA tensors run the sm_100a kernels (csrc/cuda/log_probs.cu): one pass over the logits, which are read in
their own type, and one more for the gradient; no matrix of probabilities and no copy in 32 bits.  CPU tensors
run the same formulas in torch.  Sums are kept in 32 bits; results do not depend on the order in which
thread blocks run.  First derivatives only, as for the other layer operators.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from .._native import lib as _lib
from . import _common as _c

MOST_TOP = 32


class TokenLogProbs(NamedTuple):
    """What :func:`token_log_probs` returns; ``None`` for what was not asked for."""
    log_probs: torch.Tensor
    entropy: Optional[torch.Tensor]
    top_log_probs: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


def _check(what, logits, tokens):
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: no vocabulary in logits of shape {tuple(logits.shape)}")
    if logits.dtype not in _c.TYPES and not (logits.dtype == torch.float64 and not logits.is_cuda):
        raise TypeError(f"{what}: {logits.dtype} is not supported")
    _c.same_device(what, logits, tokens)
    if tokens.dtype != torch.int64 or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"{what}: tokens are int64 of {tuple(logits.shape[:-1])}, not {tokens.dtype} of "
                         f"{tuple(tokens.shape)}")
    if logits.shape[-1] > 1 << 30 or tokens.numel() >= 1 << 31:
        raise ValueError(f"{what}: logits of {tuple(logits.shape)} are too many")


def token_log_probs(logits, tokens, *, top: int = 0, entropy: bool = True, ignore_index: int = -100) -> TokenLogProbs:
    """``log_softmax(logits)`` at ``tokens``, with the entropy of each row's distribution and its ``top``
    likeliest tokens (up to 32), likeliest first, of equal ones the lowest.

    ``logits`` [..., vocabulary]: float32, bfloat16 or float16; ``tokens`` [...], int64.  Results are float32
    (``top_tokens`` int64).  ``log_probs`` and ``entropy`` have gradients.  A token that is ``ignore_index`` has the
    log probability zero and no gradient; any other outside the vocabulary gives NaN on a GPU, an
    error on the CPU.  A row of logits that are all -inf has the log probabilities -inf, the entropy zero and no
    gradient; an infinity or a NaN among the logits makes the row's results NaN."""
    _check("token_log_probs", logits, tokens)
    top, ignore_index = int(top), int(ignore_index)
    if not 0 <= top <= min(MOST_TOP, logits.shape[-1]):
        raise ValueError(f"token_log_probs: the {top} likeliest of {logits.shape[-1]} tokens (at most {MOST_TOP})")
    run = _lib.layers().token_log_probs if logits.is_cuda else _TokenLogProbs.apply
    return TokenLogProbs(*run(logits, tokens, ignore_index, top, bool(entropy)))


def cross_entropy(logits, labels, *, ignore_index: int = -100, reduction: str = "mean"):
    """Minus the log probabilities of ``labels``: their ``"mean"`` over rows whose label is not ``ignore_index``
    (NaN if there is none), their ``"sum"``, or with ``"none"`` each by itself.  Logits, labels outside the
    vocabulary, infinities: as for :func:`token_log_probs`.  The loss is float32, its gradient has the
    logits' type."""
    _check("cross_entropy", logits, labels)
    ignore_index = int(ignore_index)
    if reduction == "none":
        return -token_log_probs(logits, labels, entropy=False, ignore_index=ignore_index).log_probs
    if reduction not in ("mean", "sum"):
        raise ValueError(f"cross_entropy: reduction {reduction!r} is none of 'mean', 'sum', 'none'")
    if logits.is_cuda:
        return _lib.layers().cross_entropy(logits, labels, ignore_index, reduction == "sum")
    lp = _TokenLogProbs.apply(logits, labels, ignore_index, 0, False)[0]
    return -lp.sum() if reduction == "sum" else -lp.sum() / (labels != ignore_index).sum()


def _result(x):
    return x if x.dtype == torch.float64 else x.float()


def _log_p(logits):
    """Log probabilities; -inf in rows that have nothing else."""
    x = _c.wide(logits)
    high = x.amax(-1, keepdim=True)
    d = x - torch.where(high == -math.inf, torch.zeros_like(high), high)
    lse = torch.log(torch.exp(d).sum(-1, keepdim=True))
    return torch.where(lse == -math.inf, d, d - lse)


def _entropy(lp):
    p = torch.exp(lp)
    return -(p * torch.where(p == 0, torch.zeros_like(lp), lp)).sum(-1)


class _TokenLogProbs(torch.autograd.Function):
    """On CPU tensors."""

    @staticmethod
    def forward(ctx, logits, tokens, ignored, top, entropy):
        there = tokens != ignored
        bad = there & ((tokens < 0) | (tokens >= logits.shape[-1]))
        if bad.any():
            raise IndexError(f"token {tokens[bad][0].item()} is not one of {logits.shape[-1]}")
        lp = _log_p(logits)
        at = torch.where(there, tokens, 0)[..., None]
        out = torch.where(there, lp.gather(-1, at)[..., 0], torch.zeros((), dtype=lp.dtype))
        h = _entropy(lp) if entropy else None
        best = torch.sort(logits, dim=-1, descending=True, stable=True).indices[..., :top] if top else None
        tops = lp.gather(-1, best) if top else None
        ctx.save_for_backward(logits, tokens)
        ctx.ignored = ignored
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(tops, best)
        return out, h, tops, best

    @staticmethod
    @_c.first_order
    def backward(ctx, dlogp, dentropy, _, __):
        if dlogp is None and dentropy is None:
            return (None,) * 5
        logits, tokens = ctx.saved_tensors
        there = tokens != ctx.ignored
        lp = _log_p(logits)
        p = torch.exp(lp)
        g = torch.zeros_like(lp[..., 0]) if dlogp is None else torch.where(there, dlogp, torch.zeros_like(dlogp))
        by = g[..., None]
        if dentropy is not None:
            by = by + dentropy[..., None] * (torch.where(p == 0, torch.zeros_like(lp), lp) + _entropy(lp)[..., None])
        d = (-p * by).scatter_add(-1, torch.where(there, tokens, 0)[..., None], g[..., None])
        some = (g != 0) if dentropy is None else (g != 0) | (dentropy != 0)
        some = some & (_c.wide(logits).amax(-1) != -math.inf)   # rows without a gradient have none, whatever they hold
        return torch.where(some[..., None], d, torch.zeros_like(d)).to(logits.dtype), None, None, None, None
