"""Bounds for each row of what the layer operators return, from the roundings on the way.

A value rounded to a type of unit roundoff u is off by at most u of itself, on average over many by
u / sqrt(3); sums of such errors add up in quadrature.  `spread` of a row is the square root of the
sum of their squares, and a row may be off by six times that (six standard deviations, for errors that are
independent), besides its own last rounding and sums of `steps` additions in 32 bits.  A row that is lost,
doubled or lacks a tile of its terms is off by a part of itself, far more."""
import math

import torch

from _layers import U, act64, attention64, linear64

SIGMAS = 6


def _bound(exact, spread, absolute, kind, steps, smallest=0.0):
    """Per row: the last rounding, the spread of the earlier ones, 32-bit sums, fp16's smallest numbers."""
    floor = math.sqrt(exact.shape[-1]) * 2.0 ** -25 if kind == torch.float16 else 0.0
    return (U[kind] * exact.norm(dim=-1) + SIGMAS * spread + steps * 2.0 ** -23 * absolute.norm(dim=-1) + floor + smallest + 1e-30)


def attention_rows(q, k, v, do, *, causal=False, mask=None, scale=None):
    """{name: (exact, bound of each row)} of out, dq, dk, dv."""
    kind = q.dtype
    want = attention64(q, k, v, do, causal=causal, mask=mask, scale=scale)
    b, sq, h, d = q.shape
    sk, hk = k.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    if mask is not None:
        k, v = (torch.where(mask[:, :, None, None], x, torch.zeros_like(x)) for x in (k, v))
    qh, gh = (t.double().transpose(1, 2) for t in (q, do))
    kh, vh = (t.double().transpose(1, 2).repeat_interleave(h // hk, 1) for t in (k, v))
    see = torch.ones(sq, sk, dtype=torch.bool, device=q.device)
    if causal:
        see = see.tril(sk - sq)
    see = see.expand(b, 1, sq, sk)
    if mask is not None:
        see = see & mask[:, None, None]
    lse = want["lse"][0]
    p = torch.exp((qh @ kh.transpose(2, 3) * scale).masked_fill(~see, -math.inf) - lse.masked_fill(lse == -math.inf, 0.0)[..., None])
    o = p @ vh
    ds = p * (gh @ vh.transpose(2, 3) - (gh * o).sum(-1, keepdim=True))
    u2 = U[kind] ** 2 / 3
    squares = lambda x: (x * x).sum(-1)  # noqa: E731
    # delta comes from the rounded result: one error for a whole row of dS
    delta2 = u2 * ((gh * o) ** 2).sum(-1)
    rows = lambda x: x.clamp(min=0).sqrt().transpose(1, 2)  # noqa: E731
    fold = lambda x: x.reshape(b, hk, h // hk, sk).sum(2)  # noqa: E731
    steps_q, steps_k = 64 + sk // 16, 64 + sq * (h // hk) // 16
    # what fp16 cannot hold of a probability, next to the largest of its row
    least = 2.0 ** -25 * (p.amax(-1) if sk else p.new_zeros(b, h, sq)) if kind == torch.float16 else p.new_zeros(b, h, sq)
    spread = {
        "out": rows(u2 * (p ** 2 @ squares(vh)[..., None])[..., 0] + least ** 2 * squares(vh).sum(-1)[..., None]),
        "dq": rows(u2 * (ds ** 2 @ squares(kh)[..., None])[..., 0] + delta2 * squares(p @ kh)) * abs(scale),
        "dk": rows(fold(((ds ** 2 * u2 + p ** 2 * delta2[..., None]).transpose(2, 3) @ squares(qh)[..., None])[..., 0])) * abs(scale),
        "dv": rows(fold(u2 * ((p ** 2).transpose(2, 3) @ squares(gh)[..., None])[..., 0]))}
    # the short kernel holds dS of all rows times one power of two, by the largest row of d_o
    small = 2.0 ** -25 * do.double().norm(dim=-1).amax().item() * abs(scale) if kind == torch.float16 and do.numel() else 0.0
    smallest = {"out": 0.0, "dv": 0.0, "dq": small * kh.norm().item(), "dk": small * qh.norm().item()}
    steps = {"out": steps_q, "dq": steps_q, "dk": steps_k, "dv": steps_k}
    return {n: (want[n][0], _bound(want[n][0], spread[n], want[n][1], kind, steps[n], smallest[n])) for n in spread}


def linear_rows(x, w, b, r, dy, activation):
    """The same of y, dx, dw; db as a matrix of one column."""
    kind = x.dtype
    want = linear64(x, w, b, r, dy, activation)
    x2, w2, dy2 = (t.double().reshape(-1, t.shape[-1]) for t in (x, w, dy))
    bias = 0 if b is None else b.double()
    p, pa = x2 @ w2.t() + bias, x2.abs() @ w2.abs().t() + (0 if b is None else bias.abs())
    g = dy2 * act64(p, activation)[1]
    u2 = U[kind] ** 2 / 3
    cast = 0.0 if w.dtype == kind else 1.0            # a 32-bit weight's own rounding
    p2 = cast * u2 * (x2 ** 2 @ (w2 ** 2).t())        # of the product, squared
    g2 = torch.zeros_like(g)
    if activation:   # the slope is taken of the rounded product, and rounded; 1.13 and 1.2 bound the first two derivatives
        smooth = 0.0 if activation == "relu" else 1.2
        g2 = u2 * g ** 2 + (smooth * dy2) ** 2 * (u2 * p ** 2 + p2)
        if activation == "relu":   # a step where the product's sign is not certain
            g2 = g2 + torch.where(p.abs() <= 8 * p2.sqrt() + 2.0 ** -20 * pa + 2.0 ** -24, dy2 ** 2, 0.0)
    m, k, n = x2.shape[0], x2.shape[1], w2.shape[0]
    norm = lambda t: t.sum(-1).sqrt()  # noqa: E731
    spread = {"y": norm(1.13 ** 2 * p2), "dx": norm((g2 + cast * u2 * g ** 2) @ w2 ** 2), "dw": norm(g2.t() @ x2 ** 2)}
    types = {"y": kind, "dx": kind, "dw": w.dtype}
    steps = {"y": 64 + k // 16, "dx": 64 + n // 16, "dw": 64 + m // 16}
    out = {name: (want[name][0], _bound(want[name][0], spread[name], want[name][1], types[name], steps[name])) for name in spread}
    if b is not None:
        exact, absolute = (t[:, None] for t in want["db"])
        out["db"] = (exact, _bound(exact, norm(g2.sum(0)[:, None]), absolute, b.dtype, 64 + m // 16))
    return out


def off(got, exact, bound):
    """The largest error of a row next to its bound; at most 1 where all are right."""
    error = (got.double().reshape(exact.shape) - exact).norm(dim=-1)
    error = torch.where(torch.isfinite(error), error, math.inf)
    return (error / bound).max().item() if error.numel() else 0.0
