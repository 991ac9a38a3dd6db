"""Layers of the models that are trained: layer norm, the matrix product with bias,
activation and residual in its epilogue, and attention, each with its gradient.

    y = layer_norm(x, weight, bias)                 y, z = layer_norm(x, weight, bias, residual=r)
    y = linear(x, weight, bias, activation="gelu")  y = linear(x, weight, bias, residual=r)
    o = attention(q, k, v, causal=True)             o = self_attention(qkv, key_mask=mask)

CUDA tensors run the sm_100a kernels (csrc/cuda/layer_norm.cu, linear.cu, attention.cu) on
the current stream of their device; CPU tensors the same formulas in torch.  Statistics,
softmax sums and products are kept in 32 bits; probabilities, their gradient and the
gradient in front of an activation are rounded to the inputs' type where they enter a matrix
product.  Results do not depend on the order in which thread blocks run: two calls with the
same inputs give the same bits.

First derivatives only: a gradient taken with ``create_graph`` refuses to be differentiated, and
forward mode is refused.

Under autocast ``linear`` and ``attention`` cast 32-bit activations to autocast's type;
``layer_norm`` keeps the type of ``x``.  Weights may be in 32 bits or in the activations'
type, and get their gradient in their own type.

The reference (mark14wu/hipress) leaves the layers to its front ends.
"""
from __future__ import annotations

import functools
import math

import torch

from .._native import lib as _lib

TYPES = (torch.float32, torch.bfloat16, torch.float16)
HALF = (torch.bfloat16, torch.float16)
ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3}


def _same_device(what, *ts):
    dev = ts[0].device
    for t in ts[1:]:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: tensors on {dev} and {t.device}")
    return dev


def _autocast(x):
    """``x`` as autocast would have a matrix product take it."""
    if x is not None and x.dtype == torch.float32 and torch.is_autocast_enabled(x.device.type):
        return x.to(torch.get_autocast_dtype(x.device.type))
    return x


def _wide(x):
    return x if x.dtype == torch.float64 else x.float()   # CPU: float64 is taken as it is


def _rows(x):
    return x.reshape(math.prod(x.shape[:-1]), x.shape[-1])   # also of no elements


class _Refused(torch.autograd.Function):
    """A value as it is, which cannot be differentiated by what it was made from."""

    @staticmethod
    def forward(ctx, x, *made_from):
        return x.view_as(x)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("a gradient of a layer operator cannot be differentiated")


def _first_order(backward):
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


# ================================================================== layer norm
def layer_norm(x, weight=None, bias=None, *, residual=None, eps: float = 1e-5):
    """Normalises the last axis of ``x``: ``(z - mean) / sqrt(var + eps) * weight + bias``.

    With ``residual`` (of ``x``'s shape and type) ``z = x + residual``, rounded to that type,
    is normalised and returned too: ``(y, z)``; both have gradients.  ``x``: float32, bfloat16
    or float16; ``weight``, ``bias``: one value per column, float32 or ``x``'s type, the same
    for both."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: no columns in a tensor of shape {tuple(x.shape)}")
    if x.dtype not in TYPES and not (x.dtype == torch.float64 and not x.is_cuda):
        raise TypeError(f"layer_norm: {x.dtype} is not supported")
    _same_device("layer_norm", x, weight, bias, residual)
    for name, w in (("weight", weight), ("bias", bias)):
        if w is None:
            continue
        if w.shape != x.shape[-1:]:
            raise ValueError(f"layer_norm: {name} of shape {tuple(w.shape)} for {x.shape[-1]} columns")
        if w.dtype not in (torch.float32, x.dtype):
            raise TypeError(f"layer_norm: {name} in {w.dtype} for x in {x.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"layer_norm: weight in {weight.dtype}, bias in {bias.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"layer_norm: a residual of {tuple(residual.shape)} {residual.dtype} for x of "
                         f"{tuple(x.shape)} {x.dtype}")
    y, z = (_lib.layers().layer_norm if x.is_cuda else _LayerNorm.apply)(x, weight, bias, residual, eps)
    return y if residual is None else (y, z)


class _LayerNorm(torch.autograd.Function):
    """On CPU tensors."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        z = x if residual is None else (_wide(x) + _wide(residual)).to(x.dtype)
        var, mean = torch.var_mean(_wide(z), -1, unbiased=False, keepdim=True)
        rstd = (var + eps).rsqrt()
        y = (_wide(z) - mean) * rstd
        if weight is not None:
            y = y * _wide(weight)
        if bias is not None:
            y = y + _wide(bias)
        ctx.save_for_backward(z, weight, mean, rstd, x, bias, residual)
        ctx.bias = None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        return y.to(x.dtype), None if residual is None else z

    @staticmethod
    @_first_order
    def backward(ctx, dy, dz):
        z, weight, mean, rstd = ctx.saved_tensors[:4]
        if dy is None and dz is None:
            return None, None, None, None, None
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        g = torch.zeros_like(mean).expand_as(z) if dy is None else _wide(dy)   # only the sum was used further on
        h = (_wide(z) - mean) * rstd
        dw = _rows(g * h).sum(0).to(weight.dtype) if need_w else None
        db = _rows(g).sum(0).to(ctx.bias) if need_b else None
        if weight is not None:
            g = g * _wide(weight)
        dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
        if dz is not None:
            dx = dx + _wide(dz)
        dx = dx.to(z.dtype)
        return dx if need_x else None, dw, db, dx if need_r else None, None


# ====================================================================== linear
def linear(x, weight, bias=None, *, activation: str | None = None, residual=None):
    """``activation(x @ weight.T + bias) + residual`` over the last axis of ``x``.

    ``activation``: None, "relu", "gelu" or "gelu_tanh".  On a GPU ``x`` and ``residual`` are
    bfloat16 or float16; ``weight`` ([out, in]) and ``bias`` float32 or ``x``'s type (a float32
    weight is rounded to it for the product; its gradient is not)."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"linear: activation {activation!r} is none of {', '.join(map(repr, ACTIVATIONS))}")
    x, residual = _autocast(x), _autocast(residual)
    _same_device("linear", x, weight, bias, residual)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: x of shape {tuple(x.shape)} and a weight of shape {tuple(weight.shape)}")
    if x.is_cuda and x.dtype not in HALF:
        raise TypeError(f"linear: the kernels take bfloat16 or float16, not {x.dtype} (use autocast)")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"linear: a bias of shape {tuple(bias.shape)} for {weight.shape[0]} outputs")
    for name, w in (("weight", weight), ("bias", bias)):
        if w is not None and w.dtype not in (torch.float32, x.dtype):
            raise TypeError(f"linear: {name} in {w.dtype} for x in {x.dtype}")
    shape = x.shape[:-1] + weight.shape[:1]
    if residual is not None and (residual.shape != shape or residual.dtype != x.dtype):
        raise ValueError(f"linear: a residual of {tuple(residual.shape)} {residual.dtype} for a result of "
                         f"{tuple(shape)} {x.dtype}")
    return (_lib.layers().linear if x.is_cuda else _Linear.apply)(x, weight, bias, residual, ACTIVATIONS[activation])


def _act(p, kind):
    if kind == 1:
        return p.clamp(min=0)
    if kind == 2:
        return p * 0.5 * (1 + torch.erf(p * math.sqrt(0.5)))
    if kind == 3:
        return 0.5 * p * (1 + torch.tanh(math.sqrt(2 / math.pi) * (p + 0.044715 * p ** 3)))
    return p


def _act_slope(p, kind):
    if kind == 1:
        return (p > 0).to(p.dtype)
    # zero and one to the last bit from here on; p may be an infinity, which its rounding made of a large value
    p = p.clamp(-64.0, 64.0)
    if kind == 2:
        return 0.5 * (1 + torch.erf(p * math.sqrt(0.5))) + p * torch.exp(-0.5 * p * p) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (p + 0.044715 * p ** 3))
    return 0.5 * (1 + t) + 0.5 * p * (1 - t * t) * c * (1 + 3 * 0.044715 * p * p)


class _Linear(torch.autograd.Function):
    """On CPU tensors."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        w = weight.to(x.dtype)
        p = _wide(x) @ _wide(w).t()
        if bias is not None:
            p = p + _wide(bias)
        y = _act(p, act)
        if residual is not None:
            y = y + _wide(residual)
        ctx.save_for_backward(x, w, p.to(x.dtype) if act else None, weight, bias, residual)
        ctx.act, ctx.types = act, (weight.dtype, None if bias is None else bias.dtype)
        return y.to(x.dtype)

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        x, w, pre = ctx.saved_tensors[:3]
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        g = _wide(dy) if pre is None else _wide(dy) * _act_slope(_wide(pre), ctx.act)
        db = _rows(g).sum(0).to(ctx.types[1]) if need_b else None
        g = _wide(g.to(x.dtype))
        dx = (g @ _wide(w)).to(x.dtype) if need_x else None
        dw = (_rows(g).t() @ _rows(_wide(x))).to(ctx.types[0]) if need_w else None
        return dx, dw, db, dy if need_r else None, None


# =================================================================== attention
def attention(q, k, v, *, causal: bool = False, key_mask=None, scale: float | None = None, return_lse: bool = False):
    """``softmax(scale q k^T) v`` for ``q`` [batch, queries, heads, dim] and ``k``, ``v``
    [batch, keys, key heads, dim], as [batch, queries, heads, dim].

    ``heads`` is a multiple of the key heads: query head ``h`` reads key head ``h // (heads //
    key heads)``.  ``causal``: query ``i`` sees the keys up to ``i + keys - queries``.
    ``key_mask`` [batch, keys], bool: the keys that may be seen; what the others hold, NaN
    among it, has no effect.  A query that sees no key gets zeros and no gradient.  ``scale``: 1 /
    sqrt(dim) unless given.  ``return_lse``: also the logarithm of each row's softmax sum
    [batch, heads, queries], float32, without a gradient (-inf where no key is seen).

    On a GPU: bfloat16 or float16, ``dim`` a multiple of 8 up to 128.  The backward pass
    computes the probabilities again, from that logarithm; there is no dropout."""
    q, k, v = _autocast(q), _autocast(k), _autocast(v)
    scale = _check_attention(q, k, v, key_mask, scale)
    o, lse = (_lib.layers().attention if q.is_cuda else _Attention.apply)(q, k, v, key_mask, causal, scale)
    return (o, lse) if return_lse else o


def self_attention(qkv, *, causal: bool = False, key_mask=None, scale: float | None = None, return_lse: bool = False):
    """:func:`attention` of ``q, k, v = qkv.unbind(2)``, [batch, length, 3, heads, dim] as one
    projection leaves them; the gradient has the same form, so that nothing is copied."""
    qkv = _autocast(qkv)
    if qkv.dim() != 5 or qkv.shape[2] != 3:
        raise ValueError(f"self_attention: [batch, length, 3, heads, dim] is wanted, not {tuple(qkv.shape)}")
    q, k, v = qkv.unbind(2)
    scale = _check_attention(q, k, v, key_mask, scale)
    if qkv.is_cuda:
        o, lse = _lib.layers().self_attention(qkv, key_mask, causal, scale)
    else:
        o, lse = _Attention.apply(q, k, v, key_mask, causal, scale)
    return (o, lse) if return_lse else o


def _check_attention(q, k, v, mask, scale):
    _same_device("attention", q, k, v, mask)
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError("attention: [batch, length, heads, dim] is wanted, k and v alike: got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if not q.dtype == k.dtype == v.dtype:
        raise TypeError(f"attention: q, k, v in {q.dtype}, {k.dtype}, {v.dtype}")
    if k.shape[2] < 1 or q.shape[2] < 1 or q.shape[2] % k.shape[2]:
        raise ValueError(f"attention: {q.shape[2]} heads over {k.shape[2]} key heads")
    if q.shape[3] < 1:
        raise ValueError("attention: heads without a dimension")
    if q.is_cuda:
        if q.dtype not in HALF:
            raise TypeError(f"attention: the kernels take bfloat16 or float16, not {q.dtype} (use autocast)")
        if q.shape[3] % 8 or q.shape[3] > 128:
            raise ValueError(f"attention: head dimension {q.shape[3]} is no multiple of 8 up to 128")
        if q.shape[0] > 65535 or q.shape[2] > 65535:
            raise ValueError(f"attention: more than 65535 sequences or heads: {tuple(q.shape)}")
    if mask is not None and (mask.dtype != torch.bool or mask.shape != k.shape[:2]):
        raise ValueError(f"attention: key_mask is bool of {tuple(k.shape[:2])}, not {mask.dtype} of {tuple(mask.shape)}")
    scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"attention: scale {scale}")
    return scale


def _hidden(q, k, mask, causal):
    sq, sk = q.shape[1], k.shape[1]
    seen = torch.ones(sq, sk, dtype=torch.bool, device=q.device)
    if causal:
        seen = seen.tril(sk - sq)
    seen = seen[None, None]
    return seen if mask is None else seen & mask[:, None, None]


def _cpu_heads(q, k, v, mask):
    """[batch, heads, length, dim], shared key heads repeated, masked keys and values zero."""
    if mask is not None:
        k, v = (torch.where(mask[:, :, None, None], x, torch.zeros((), dtype=x.dtype)) for x in (k, v))
    group = q.shape[2] // k.shape[2]
    return (_wide(q).transpose(1, 2), *(_wide(x).transpose(1, 2).repeat_interleave(group, 1) for x in (k, v)))


class _Attention(torch.autograd.Function):
    """On CPU tensors."""

    @staticmethod
    def forward(ctx, q, k, v, mask, causal, scale):
        (b, sq, h, _), sk = q.shape, k.shape[1]
        qh, kh, vh = _cpu_heads(q, k, v, mask)
        s = (qh @ kh.transpose(2, 3) * scale).masked_fill(~_hidden(q, k, mask, causal), -math.inf)
        lse = torch.logsumexp(s, -1) if sk else s.new_full((b, h, sq), -math.inf)
        p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[..., None])
        o = (p @ vh).transpose(1, 2).to(q.dtype).contiguous()
        ctx.save_for_backward(q, k, v, o, lse, mask)
        ctx.causal, ctx.scale = causal, scale
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @_first_order
    def backward(ctx, do, _):
        if do is None:
            return (None,) * 6
        q, k, v, o, lse, mask = ctx.saved_tensors
        (b, _, h, d), sk, hk = q.shape, k.shape[1], k.shape[2]
        qh, kh, vh = _cpu_heads(q, k, v, mask)
        g, oh = _wide(do).transpose(1, 2), _wide(o).transpose(1, 2)
        s = (qh @ kh.transpose(2, 3) * ctx.scale).masked_fill(~_hidden(q, k, mask, ctx.causal), -math.inf)
        p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[..., None])
        ds = p * (g @ vh.transpose(2, 3) - (g * oh).sum(-1, keepdim=True)) * ctx.scale
        group = lambda x: x.view(b, hk, h // hk, sk, d).sum(2)  # noqa: E731
        out = ds @ kh, group(ds.transpose(2, 3) @ qh), group(p.transpose(2, 3) @ g)
        need = ctx.needs_input_grad
        return (*(x.transpose(1, 2).to(q.dtype) if n else None for x, n in zip(out, need)), None, None, None)
