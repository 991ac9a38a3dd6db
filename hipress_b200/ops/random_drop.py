"""Dropout whose mask is never stored: which elements are kept is a function of a seed, the call's number
under that seed, and the element's place.

    y = dropout(x, 0.1, seed=seed, site=3)                 y = dropout(x, 0.1, seed=seed, residual=r)

The backward pass computes the same bits again, and so does a second forward pass with the same seed
(activation checkpointing, a replayed step).  ``layer_norm``, ``attention`` and ``self_attention`` take the same
arguments.

``seed``: an int, or an int64 tensor of one element on the device of ``x``, which is read when the kernel
runs.  A step that is captured into a CUDA graph moves such a tensor on (``seed.add_(1)``) and gets another
mask at every replay; between a forward pass and its backward pass it must not change (autograd raises if it
has).  ``site``: tells the calls under one seed apart, 0 .. 2^32 - 1.

The definition: elements are counted in their logical order (attention probabilities as [batch, heads, queries,
keys], the keys rounded up to a multiple of 32), 32 to a word.  Word ``w`` has 16 random words, the results of
Philox4x32 with 7 rounds under the key ``seed`` for the counters ``(w mod 2^32, w div 2^32, site, 0 .. 3)``.  Bit
``i`` of the j-th is bit j of a number of 16 bits for element ``32 w + i``; the element is kept where
that number is at least ``2^16 - t``, ``t = (1 - p) 2^16`` rounded to 1 .. 2^16, and then multiplied by ``2^16 /
t``.  So ``p`` is met to 2^-17, and the expectation exactly.  A dropped element is zero whatever it was.

CUDA tensors run the sm_100a kernels (csrc/cuda/dropout.cu, philox.cuh), CPU tensors the same definition
in torch.
"""
from __future__ import annotations

import torch

from .._native import lib as _lib
from . import _common as _c


def random_args(what: str, x: torch.Tensor, p: float, seed, site: int):
    """``(seed tensor or None, seed, site, t)`` of a dropout of ``x``; ``t`` is 0 where nothing is dropped."""
    p = float(p)
    if not 0.0 <= p < 1.0:
        raise ValueError(f"{what}: a dropout probability of {p} is not in [0, 1)")
    if not 0 <= int(site) < 2 ** 32:
        raise ValueError(f"{what}: site {site} is not in [0, 2^32)")
    keep = max(1, round((1.0 - p) * 65536))
    if keep == 65536:
        return None, 0, 0, 0
    if seed is None:
        raise ValueError(f"{what}: a dropout wants a seed")
    if not isinstance(seed, torch.Tensor):
        seed = int(seed)
        if not -2 ** 63 <= seed < 2 ** 64:
            raise ValueError(f"{what}: seed {seed} has more than 64 bits")
        return None, seed - 2 ** 64 if seed >= 2 ** 63 else seed, int(site), keep
    if seed.dtype != torch.int64 or seed.numel() != 1:
        raise TypeError(f"{what}: a seed is an int or an int64 tensor of one element, not {seed.dtype} of "
                        f"{tuple(seed.shape)}")
    if seed.device != x.device:
        raise ValueError(f"{what}: tensors on {x.device} and {seed.device}")
    return seed, 0, int(site), keep


_WORD = 0xFFFFFFFF


def _philox(c, k0, k1):
    x0, x1, x2, x3 = c
    for _ in range(7):
        a, b = x0 * 0xD2511F53, x2 * 0xCD9E8D57    # int64 wraps; the bits are those of the product
        x0, x1, x2, x3 = ((b >> 32) & _WORD) ^ x1 ^ k0, b & _WORD, ((a >> 32) & _WORD) ^ x3 ^ k1, a & _WORD
        k0, k1 = (k0 + 0x9E3779B9) & _WORD, (k1 + 0xBB67AE85) & _WORD
    return x0, x1, x2, x3


def _kept(words: int, random) -> torch.Tensor:
    """Whether each of the first ``32 words`` elements is kept; on the CPU."""
    seed_at, seed, site, keep = random
    if seed_at is not None:
        seed = int(seed_at)
    w = torch.arange(words)
    m = torch.zeros_like(w)
    for call in range(4):
        c = w & _WORD, w >> 32, torch.full_like(w, site), torch.full_like(w, call)
        for j, r in enumerate(_philox(c, seed & _WORD, (seed >> 32) & _WORD)):
            m = m | r if keep >> (4 * call + j) & 1 else m & r
    return (m[:, None] >> torch.arange(32) & 1).bool().flatten()


def kept_elements(shape, random) -> torch.Tensor:
    n = torch.Size(shape).numel()
    return _kept((n + 31) // 32, random)[:n].view(shape)


def kept_probabilities(b: int, h: int, sq: int, sk: int, random) -> torch.Tensor:
    words = (sk + 31) // 32
    return _kept(b * h * sq * words, random).view(b, h, sq, 32 * words)[..., :sk]


def dropped(x, kept, keep: int):
    """``x`` in wide numbers: where it is not kept zero, whatever it is."""
    return torch.where(kept, x * (65536 / keep), torch.zeros((), dtype=x.dtype))


class _Dropout(torch.autograd.Function):
    """On CPU tensors."""

    @staticmethod
    def forward(ctx, x, residual, *random):
        ctx.save_for_backward(x, residual, random[0])
        ctx.random = random[1:]
        y = dropped(_c.wide(x), kept_elements(x.shape, random), random[3])
        return (y if residual is None else y + _c.wide(residual)).to(x.dtype)

    @staticmethod
    @_c.first_order
    def backward(ctx, dy):
        random = (ctx.saved_tensors[2], *ctx.random)
        need_x, need_r = ctx.needs_input_grad[:2]
        dx = dropped(_c.wide(dy), kept_elements(dy.shape, random), random[3]).to(dy.dtype) if need_x else None
        return dx, dy if need_r else None, None, None, None, None


def dropout(x, p: float, *, seed=None, site: int = 0, residual=None):
    """``x`` with elements dropped with the probability ``p`` and the others multiplied by 1 / (1 - p); plus
    ``residual`` (of ``x``'s shape and type), in the same pass.  ``x``: float32, bfloat16 or float16.  See
    the module for ``seed`` and ``site``."""
    if x.dtype not in _c.TYPES and not (x.dtype == torch.float64 and not x.is_cuda):
        raise TypeError(f"dropout: {x.dtype} is not supported")
    _c.same_device("dropout", x, residual)
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"dropout: a residual of {tuple(residual.shape)} {residual.dtype} for x of "
                         f"{tuple(x.shape)} {x.dtype}")
    random = random_args("dropout", x, p, seed, site)
    if not random[3]:
        return x.clone() if residual is None else x + residual
    if x.is_cuda:
        return _lib.layers().dropout(x, residual, *random)
    return _Dropout.apply(x, residual, *random)
