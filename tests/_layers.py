"""The layer operators in 64 bits, for their tests: results and, for each, the same sums over
absolute values.  An error bound is a number of roundings times that: a value that is rounded
to a type of unit roundoff u on its way into a sum of products changes the sum by at most u
times the sum of the products' absolute values."""
import math

import torch

# unit roundoff: half the distance between neighbours of 1
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float64: 2.0 ** -53}


def close(got, want, scale, roundings, kind, what, steps=64):
    """2-norms: ``roundings`` roundings to ``kind``, and sums of ``steps`` additions in 32 bits.
    A rounding to fp16 may also lose up to 2^-25, half its smallest number."""
    bound = (roundings * U[kind] + steps * 2.0 ** -23) * scale.double().norm() + \
        (math.sqrt(max(got.numel(), 1)) * 2.0 ** -25 * roundings if kind == torch.float16 else 0.0)
    err = (got.double() - want).norm()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all() or not torch.isfinite(want).all(), f"{what}: not finite"
    assert err <= bound, f"{what}: off by {err.item():.3g}, bound {bound.item():.3g}, norm {want.norm().item():.3g}"


def norm64(z, w, b, dy, dz, eps):
    z, dy = z.double(), dy.double()
    w = torch.ones(z.shape[-1], dtype=torch.float64, device=z.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mean = z.mean(-1, keepdim=True)
    s = 1 / torch.sqrt(((z - mean) ** 2).mean(-1, keepdim=True) + eps)
    h = (z - mean) * s
    # z - mean cancels where the mean is large: 32 bits of z, not of the difference
    ha = h.abs() + s * (z.abs() + mean.abs()) * 2.0 ** -4
    g = dy * w
    dx = s * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    ga = g.abs()
    dxa = s * (ga + ga.mean(-1, keepdim=True) + ha * (ga * ha).mean(-1, keepdim=True))
    if dz is not None:
        dx, dxa = dx + dz.double(), dxa + dz.double().abs()
    over_rows = lambda t: t.reshape(-1, t.shape[-1]).sum(0)  # noqa: E731
    return {"y": (h * w + b, ha * w.abs() + b.abs()), "dx": (dx, dxa),
            "dw": (over_rows(dy * h), over_rows(dy.abs() * ha)), "db": (over_rows(dy), over_rows(dy.abs()))}


def act64(p, kind):
    if kind is None:
        return p, torch.ones_like(p)
    if kind == "relu":
        return p.clamp(min=0), (p > 0).double()
    if kind == "gelu":
        c = 0.5 * torch.special.erfc(-p / math.sqrt(2))
        return p * c, c + p * torch.exp(-p * p / 2) / math.sqrt(2 * math.pi)
    u = math.sqrt(2 / math.pi) * (p + 0.044715 * p ** 3)
    g = torch.sigmoid(2 * u)
    return p * g, g + p * g * (1 - g) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * p * p)


def linear64(x, w, b, r, dy, kind):
    x, w, dy = (t.double().reshape(-1, t.shape[-1]) for t in (x, w, dy))
    p, pa = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        p, pa = p + b.double(), pa + b.double().abs()
    y, slope = act64(p, kind)
    ya = pa * 1.13   # no activation here is steeper than 1.13
    if r is not None:
        y, ya = y + r.double().reshape(y.shape), ya + r.double().abs().reshape(y.shape)
    g = dy * slope
    ga = dy.abs() * 1.13 if kind else dy.abs()
    return {"y": (y, ya), "dx": (g @ w, ga @ w.abs()), "dw": (g.t() @ x, ga.t() @ x.abs()), "db": (g.sum(0), ga.sum(0))}


def attention64(q, k, v, do, *, causal, mask, scale=None):
    b, sq, h, d = q.shape
    sk, hk = k.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    if mask is not None:   # what a masked key holds does not matter
        k = torch.where(mask[:, :, None, None], k, torch.zeros_like(k))
        v = torch.where(mask[:, :, None, None], v, torch.zeros_like(v))
    q, do = (t.double().transpose(1, 2) for t in (q, do))
    k, v = (t.double().transpose(1, 2).repeat_interleave(h // hk, 1) for t in (k, v))
    see = torch.ones(sq, sk, dtype=torch.bool, device=q.device)
    if causal:
        see = see.tril(sk - sq)
    see = see.expand(b, 1, sq, sk)
    if mask is not None:
        see = see & mask[:, None, None]
    s = (q @ k.transpose(2, 3) * scale).masked_fill(~see, -math.inf)
    top = s.amax(-1, keepdim=True) if sk else s.new_full((b, h, sq, 1), -math.inf)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    lse = (top + torch.log(total))[..., 0]
    p = e / torch.where(total == 0, 1.0, total)
    o = p @ v
    dp = do @ v.transpose(2, 3)
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dsa = p * (do.abs() @ v.abs().transpose(2, 3) + (do.abs() * (p @ v.abs())).sum(-1, keepdim=True))
    fold = lambda t: t.reshape(b, hk, h // hk, sk, d).sum(2).transpose(1, 2)  # noqa: E731
    back = lambda t: t.transpose(1, 2)  # noqa: E731
    return {"out": (back(o), back(p @ v.abs())), "lse": (lse, None),
            "dq": (back(ds @ k) * scale, back(dsa @ k.abs()) * abs(scale)),
            "dk": (fold(ds.transpose(2, 3) @ q) * scale, fold(dsa.transpose(2, 3) @ q.abs()) * abs(scale)),
            "dv": (fold(p.transpose(2, 3) @ do), fold(p.transpose(2, 3) @ do.abs()))}
