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

Under autocast ``linear`` and ``attention`` cast 32-bit activations to autocast's type;
``layer_norm`` keeps the type of ``x``.  Weights may be in 32 bits or in the activations'
type, and get their gradient in their own type.

The reference (mark14wu/hipress) leaves the layers to its front ends.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from .._native import lib as _lib

TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
HALF = (torch.bfloat16, torch.float16)
ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3}


def _p(t):
    return None if t is None else t.data_ptr()


def _call(name, device, *args):
    F = _lib.fast_cuda()
    if device.index == _lib.current_device():
        rc = getattr(F, name)(*args, _lib.stream_ptr())
    else:
        with torch.cuda.device(device):
            rc = getattr(F, name)(*args, _lib.stream_ptr())
    if rc:
        _lib.check(rc, name)


def _scratch(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _same_device(what, *ts):
    dev = ts[0].device
    for t in ts[1:]:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: tensors on {dev} and {t.device}")
    return dev


def _differentiable(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _autocast(x):
    """``x`` as autocast would have a matrix product take it."""
    if x is not None and x.dtype == torch.float32 and torch.is_autocast_enabled(x.device.type):
        return x.to(torch.get_autocast_dtype(x.device.type))
    return x


def _wide(x):
    return x if x.dtype == torch.float64 else x.float()   # CPU: float64 is taken as it is


def _rows(x):
    """``x`` as a matrix whose rows are dense; a copy only where there is no such view."""
    x = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _pitch(x):
    # of one row there is no second to be reached, and its stride may be anything
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


# ================================================================== layer norm
def layer_norm(x, weight=None, bias=None, *, residual=None, eps: float = 1e-5):
    """Normalises the last axis of ``x``: ``(z - mean) / sqrt(var + eps) * weight + bias``.

    With ``residual`` (of ``x``'s shape and type) ``z = x + residual``, rounded to that type,
    is normalised and returned too: ``(y, z)``; both have gradients.  ``x``: float32, bfloat16
    or float16; ``weight``, ``bias``: one value per column, float32 or ``x``'s type, the same
    for both."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: no columns in a tensor of shape {tuple(x.shape)}")
    if x.dtype not in TYPE and not (x.dtype == torch.float64 and not x.is_cuda):
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
    if _differentiable(x, weight, bias, residual):
        y, z = _LayerNorm.apply(x, weight, bias, residual, eps)
    else:
        y, z, _, _, _ = _norm_forward(x, weight, bias, residual, eps)
    return y if residual is None else (y, z)


def _norm_forward(x, weight, bias, residual, eps):
    """y, z (None without a residual), the rows that were normalised, and their statistics."""
    x2 = _rows(x)
    r2 = None if residual is None else _rows(residual)
    rows, cols = x2.shape
    if not x.is_cuda:
        z2 = x2 if r2 is None else (_wide(x2) + _wide(r2)).to(x.dtype)
        var, mean = torch.var_mean(_wide(z2), 1, unbiased=False)
        rstd = (var + eps).rsqrt()
        y = (_wide(z2) - mean[:, None]) * rstd[:, None]
        if weight is not None:
            y = y * _wide(weight)
        if bias is not None:
            y = y + _wide(bias)
        return (y.to(x.dtype).view(x.shape), None if r2 is None else z2.view(x.shape), z2, mean, rstd)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    z = None if r2 is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty(2, rows, dtype=torch.float32, device=x.device)
    w = weight if weight is not None else bias
    _call("norm_forward", x.device, x2.data_ptr(), _p(r2), _p(_dense(weight)), _p(_dense(bias)), y.data_ptr(), _p(z),
          stats.data_ptr(), stats.data_ptr() + 4 * rows, rows, cols, _pitch(x2), 0 if r2 is None else _pitch(r2),
          TYPE[x.dtype], 0 if w is None else TYPE[w.dtype], float(eps))
    return y, z, (x2 if z is None else z.view(rows, cols)), stats[0], stats[1]


def _dense(w):
    return w if w is None or w.is_contiguous() else w.contiguous()


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        y, z, rows, mean, rstd = _norm_forward(x, weight, bias, residual, eps)
        ctx.save_for_backward(rows, weight, mean, rstd)
        ctx.shape, ctx.bias, ctx.set_z = x.shape, None if bias is None else bias.dtype, z is not None
        ctx.set_materialize_grads(False)
        return y, z

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dz):
        z, weight, mean, rstd = ctx.saved_tensors
        if dy is None and dz is None:
            return None, None, None, None, None
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        if dy is None:   # only the sum was used further on
            zero = lambda need, w: torch.zeros(z.shape[1], dtype=w, device=z.device) if need else None  # noqa: E731
            return (dz if need_x else None, zero(need_w, weight.dtype if need_w else None), zero(need_b, ctx.bias),
                    dz if need_r else None, None)
        dy2, dz2 = _rows(dy), None if dz is None else _rows(dz)
        rows, cols = z.shape
        if not z.is_cuda:
            h, g = (_wide(z) - mean[:, None]) * rstd[:, None], _wide(dy2)
            dw = (g * h).sum(0).to(weight.dtype) if need_w else None
            db = g.sum(0).to(ctx.bias) if need_b else None
            if weight is not None:
                g = g * _wide(weight)
            dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
            if dz2 is not None:
                dx = dx + _wide(dz2)
            dx = dx.to(z.dtype).view(ctx.shape)
        else:
            wtype = weight.dtype if weight is not None else ctx.bias
            dx = torch.empty(ctx.shape, dtype=z.dtype, device=z.device) if need_x or need_r else None
            dw = torch.empty(cols, dtype=wtype, device=z.device) if need_w else None
            db = torch.empty(cols, dtype=wtype, device=z.device) if need_b else None
            ws = _scratch(_lib.fast_cuda().norm_workspace(rows, cols) if need_w or need_b else 0, z.device)
            _call("norm_backward", z.device, z.data_ptr(), dy2.data_ptr(), _p(dz2), _p(_dense(weight)), mean.data_ptr(),
                  rstd.data_ptr(), _p(dx), _p(dw), _p(db), _p(ws), rows, cols, _pitch(z), _pitch(dy2),
                  0 if dz2 is None else _pitch(dz2), TYPE[z.dtype], 0 if wtype is None else TYPE[wtype])
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
    if _differentiable(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, residual, activation)
    return _linear_forward(x, weight, bias, residual, activation, False)[0]


def _operand(x, dtype):
    """A matrix a kernel can fetch by tiles: of that type, rows on 16-byte boundaries."""
    if x.dtype == dtype and x.stride(1) == 1 and x.data_ptr() % 16 == 0 and (_pitch(x) % 8 == 0 or x.shape[0] == 1):
        return x
    rows, cols = x.shape
    return torch.empty(rows, (cols + 7) // 8 * 8, dtype=dtype, device=x.device)[:, :cols].copy_(x)


def _product(a, b, m, n, k, a_k, b_k, out_type, *, bias=None, residual=None, pre=None, act=0):
    y = torch.empty(m, n, dtype=out_type, device=a.device)
    ws = _scratch(_lib.fast_cuda().product_workspace(m, n, k), a.device)
    _call("product", a.device, a.data_ptr(), b.data_ptr(), _p(bias), _p(residual), y.data_ptr(), _p(pre), _p(ws),
          m, n, k, _pitch(a), _pitch(b), n, 0 if residual is None else _pitch(residual), a_k, b_k,
          TYPE[a.dtype], TYPE[out_type], 0 if bias is None else TYPE[bias.dtype], act)
    return y


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
    if kind == 2:
        return 0.5 * (1 + torch.erf(p * math.sqrt(0.5))) + p * torch.exp(-0.5 * p * p) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (p + 0.044715 * p ** 3))
    return 0.5 * (1 + t) + 0.5 * p * (1 - t * t) * c * (1 + 3 * 0.044715 * p * p)


def _linear_forward(x, weight, bias, residual, activation, keep):
    """y and, with ``keep``, what the backward pass reads: x and the weight as the product
    took them, and the product in front of the activation."""
    act = ACTIVATIONS[activation]
    x2 = _rows(x)
    r2 = None if residual is None else _rows(residual)
    m, k = x2.shape
    n = weight.shape[0]
    shape = x.shape[:-1] + (n,)
    if not x.is_cuda:
        w = weight if x.dtype == weight.dtype else weight.to(x.dtype)
        p = _wide(x2) @ _wide(w).t()
        if bias is not None:
            p = p + _wide(bias)
        y = _act(p, act)
        if r2 is not None:
            y = y + _wide(r2)
        return y.to(x.dtype).view(shape), x2, w, (p.to(x.dtype) if act and keep else None)
    a, w = _operand(x2, x.dtype), _operand(weight.detach(), x.dtype)
    pre = torch.empty(m, n, dtype=x.dtype, device=x.device) if act and keep else None
    y = _product(a, w, m, n, k, 1, 1, x.dtype, bias=_dense(bias), residual=r2, pre=pre, act=act)
    return y.view(shape), a, w, pre


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        y, a, w, pre = _linear_forward(x, weight, bias, residual, activation, True)
        ctx.save_for_backward(a, w, pre)
        ctx.act, ctx.shape = ACTIVATIONS[activation], x.shape
        ctx.types = weight.dtype, None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, pre = ctx.saved_tensors
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        dy2 = _rows(dy)
        (m, k), n, act = x.shape, w.shape[0], ctx.act
        wtype, btype = ctx.types
        dx = dw = db = None
        if not x.is_cuda:
            g = _wide(dy2) if pre is None else _wide(dy2) * _act_slope(_wide(pre), act)
            if need_b:
                db = g.sum(0).to(btype)
            g = _wide(g.to(x.dtype))
            if need_x:
                dx = (g @ _wide(w)).to(x.dtype).view(ctx.shape)
            if need_w:
                dw = (g.t() @ _wide(x)).to(wtype)
        else:
            g = dy2
            # rows that a tile copy cannot start at are laid out anew, as is what an activation changes
            ragged = dy2.data_ptr() % 16 != 0 or (_pitch(dy2) % 8 != 0 and m > 1)
            if act or ragged:
                g = torch.empty(m, (n + 7) // 8 * 8, dtype=x.dtype, device=x.device)[:, :n]
            if g is not dy2 or need_b:
                if need_b:
                    db = torch.empty(n, dtype=btype, device=x.device)
                ws = _scratch(_lib.fast_cuda().slope_workspace(m, n) if need_b else 0, x.device)
                _call("slope", x.device, dy2.data_ptr(), _p(pre), None if g is dy2 else g.data_ptr(), _p(db), _p(ws),
                      m, n, _pitch(dy2), n, _pitch(g), TYPE[x.dtype], 0 if btype is None else TYPE[btype], act)
            if need_x:
                dx = _product(g, w, m, k, n, 1, 0, x.dtype).view(ctx.shape)
            if need_w:
                dw = _product(g, x, n, k, m, 0, 0, wtype)
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
    if _differentiable(q, k, v):
        o, lse = _Attention.apply(q, k, v, key_mask, causal, scale)
    else:
        o, lse = _attention_forward(q, k, v, key_mask, causal, scale)
    return (o, lse) if return_lse else o


def self_attention(qkv, *, causal: bool = False, key_mask=None, scale: float | None = None, return_lse: bool = False):
    """:func:`attention` of ``q, k, v = qkv.unbind(2)``, [batch, length, 3, heads, dim] as one
    projection leaves them; the gradient has the same form, so that nothing is copied."""
    qkv = _autocast(qkv)
    if qkv.dim() != 5 or qkv.shape[2] != 3:
        raise ValueError(f"self_attention: [batch, length, 3, heads, dim] is wanted, not {tuple(qkv.shape)}")
    scale = _check_attention(*qkv.unbind(2), key_mask, scale)
    if _differentiable(qkv):
        o, lse = _SelfAttention.apply(qkv, key_mask, causal, scale)
    else:
        o, lse = _attention_forward(*qkv.unbind(2), key_mask, causal, scale)
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


def _tileable(x):
    """``x`` itself where tiles of it can be fetched (the last axis dense, everything on 16-byte
    boundaries), else a copy."""
    if x.stride(3) == 1 and x.data_ptr() % 16 == 0 and not (x.stride(0) | x.stride(1) | x.stride(2)) % 8 and \
            min(x.stride()) > 0:
        return x
    return x.contiguous() if not x.is_contiguous() else x.clone()


def _strides(x):
    return x.stride()[:3]


_NO_STRIDES = (0, 0, 0)


def _mask(mask):
    return mask if mask is None or mask.stride(1) == 1 else mask.contiguous()


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


def _attention_forward(q, k, v, mask, causal, scale):
    (b, sq, h, d), sk = q.shape, k.shape[1]
    if not q.is_cuda:
        qh, kh, vh = _cpu_heads(q, k, v, mask)
        s = (qh @ kh.transpose(2, 3) * scale).masked_fill(~_hidden(q, k, mask, causal), -math.inf)
        lse = torch.logsumexp(s, -1) if sk else s.new_full((b, h, sq), -math.inf)
        p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[..., None])
        return (p @ vh).transpose(1, 2).to(q.dtype).contiguous(), lse
    o = torch.empty(b, sq, h, d, dtype=q.dtype, device=q.device)
    lse = torch.empty(b, h, sq, dtype=torch.float32, device=q.device)
    q, k, v, mask = _tileable(q), _tileable(k), _tileable(v), _mask(mask)
    _call("attention_forward", q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), _p(mask),
          None, None, None, None, None, b, sq, sk, h, k.shape[2], d, *_strides(q), *_strides(k), *_strides(v),
          *_strides(o), *_NO_STRIDES, *_NO_STRIDES, *_NO_STRIDES, *_NO_STRIDES, 0 if mask is None else mask.stride(0),
          TYPE[q.dtype], 1 if causal else 0, scale)
    return o, lse


def _attention_backward(q, k, v, o, lse, do, mask, causal, scale, dq, dk, dv):
    (b, sq, h, d), sk, hk = q.shape, k.shape[1], k.shape[2]
    if not q.is_cuda:
        qh, kh, vh = _cpu_heads(q, k, v, mask)
        g, oh = _wide(do).transpose(1, 2), _wide(o).transpose(1, 2)
        s = (qh @ kh.transpose(2, 3) * scale).masked_fill(~_hidden(q, k, mask, causal), -math.inf)
        p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[..., None])
        ds = p * (g @ vh.transpose(2, 3) - (g * oh).sum(-1, keepdim=True)) * scale
        group = lambda x: x.view(b, hk, h // hk, sk, d).sum(2).transpose(1, 2)  # noqa: E731
        dq.copy_((ds @ kh).transpose(1, 2))
        dk.copy_(group(ds.transpose(2, 3) @ qh))
        dv.copy_(group(p.transpose(2, 3) @ g))
        return
    q, k, v, do, mask = _tileable(q), _tileable(k), _tileable(v), _tileable(do), _mask(mask)
    delta = torch.empty(b, h, 2, (sq + 127) // 128 * 128, dtype=torch.float32, device=q.device)
    _call("attention_backward", q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), _p(mask),
          do.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), delta.data_ptr(), b, sq, sk, h, hk, d,
          *_strides(q), *_strides(k), *_strides(v), *_strides(o), *_strides(do), *_strides(dq), *_strides(dk),
          *_strides(dv), 0 if mask is None else mask.stride(0), TYPE[q.dtype], 1 if causal else 0, scale)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, causal, scale):
        o, lse = _attention_forward(q, k, v, mask, causal, scale)
        ctx.save_for_backward(q, k, v, o, lse, mask)
        ctx.causal, ctx.scale = causal, scale
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, do, _):
        if do is None:
            return (None,) * 6
        q, k, v, o, lse, mask = ctx.saved_tensors
        dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v))
        _attention_backward(q, k, v, o, lse, do, mask, ctx.causal, ctx.scale, dq, dk, dv)
        need = ctx.needs_input_grad
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, None, None


class _SelfAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, mask, causal, scale):
        o, lse = _attention_forward(*qkv.unbind(2), mask, causal, scale)
        ctx.save_for_backward(qkv, o, lse, mask)
        ctx.causal, ctx.scale = causal, scale
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, do, _):
        if do is None:
            return (None,) * 4
        qkv, o, lse, mask = ctx.saved_tensors
        dqkv = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        _attention_backward(*qkv.unbind(2), o, lse, do, mask, ctx.causal, ctx.scale, *dqkv.unbind(2))
        return dqkv, None, None, None
