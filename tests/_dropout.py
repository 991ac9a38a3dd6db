"""Dropout in the layer operators' tests: the generator in plain integers, and the formulas in 64 bits with
what they are bounded by (tests/_layers.py says how)."""
import math

import torch

M32 = 0xFFFFFFFF


def philox(counter, key, rounds):
    """Philox4x32 as its paper defines it."""
    x, (k0, k1) = list(counter), key
    for _ in range(rounds):
        a, b = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [(b >> 32) ^ x[1] ^ k0, b & M32, (a >> 32) ^ x[3] ^ k1, a & M32]
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    return x


def kept_count(p):
    return max(1, round((1 - p) * 65536))


def kept_bits(word, seed, site, t):
    """The 32 elements of a word, each by its number of 16 bits."""
    seed %= 2 ** 64
    u = [0] * 32
    for call in range(4):
        for j, r in enumerate(philox((word & M32, word >> 32, site, call), (seed & M32, seed >> 32), 7)):
            for i in range(32):
                u[i] |= (r >> i & 1) << (4 * call + j)
    return [x >= 65536 - t for x in u]


def kept(shape, p, seed, site, device="cpu"):
    """Of a tensor's elements; vectorised, tested against kept_bits()."""
    from hipress_b200.ops.random_drop import kept_elements
    return kept_elements(shape, (None, seed, site, kept_count(p))).to(device)


def kept_probabilities(b, h, sq, sk, p, seed, site, device="cpu"):
    from hipress_b200.ops.random_drop import kept_probabilities as f
    return f(b, h, sq, sk, (None, seed, site, kept_count(p))).to(device)


def attention64(q, k, v, do, *, causal, mask, kept, up, scale=None):
    """With ``kept`` probabilities times ``up``; sums over absolute values beside the results."""
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
    p = e / torch.where(total == 0, 1.0, total)
    m = kept.double() * up
    pm = p * m
    o = pm @ v
    oa = pm @ v.abs()
    dp = (do @ v.transpose(2, 3)) * m
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    dsa = p * ((do.abs() @ v.abs().transpose(2, 3)) * m + (do.abs() * oa).sum(-1, keepdim=True))
    fold = lambda t: t.reshape(b, hk, h // hk, sk, d).sum(2).transpose(1, 2)  # noqa: E731
    back = lambda t: t.transpose(1, 2)  # noqa: E731
    return {"out": (back(o), back(oa)), "lse": ((top + torch.log(total))[..., 0], None),
            "dq": (back(ds @ k) * scale, back(dsa @ k.abs()) * abs(scale)),
            "dk": (fold(ds.transpose(2, 3) @ q) * scale, fold(dsa.transpose(2, 3) @ q.abs()) * abs(scale)),
            "dv": (fold(pm.transpose(2, 3) @ do), fold(pm.transpose(2, 3) @ do.abs()))}


def log_probs64(x, tokens, ignored=-100):
    """(log probabilities of all, of the tokens, entropy); a row of -inf: -inf, -inf (or 0), 0."""
    x = x.double()
    top = x.amax(-1, keepdim=True)
    none = top == -math.inf
    d = x - torch.where(none, torch.zeros_like(top), top)
    lp = d - torch.where(none, torch.zeros_like(top), torch.exp(d).sum(-1, keepdim=True).log())
    there = tokens != ignored
    at = torch.where(there, tokens, 0)[..., None]
    got = torch.where(there, lp.gather(-1, at)[..., 0], 0.0)
    p = torch.exp(lp)
    return lp, got, -(p * torch.where(p == 0, 0.0, lp)).sum(-1)


def log_probs64_gradient(x, tokens, g, h, ignored=-100):
    """And its bound's scale, element by element."""
    lp, _, entropy = log_probs64(x, tokens, ignored)
    p = torch.exp(lp)
    there = tokens != ignored
    g = torch.where(there, g.double(), 0.0)[..., None]
    h = h.double()[..., None]
    z = torch.where(p == 0, 0.0, lp)
    d, da = -p * (g + h * (z + entropy[..., None])), p * (g.abs() + h.abs() * (z.abs() + entropy[..., None]))
    at = torch.where(there, tokens, 0)[..., None]
    some = (x.amax(-1, keepdim=True) != -math.inf).double()   # rows of -inf have no gradient
    return d.scatter_add(-1, at, g) * some, da.scatter_add(-1, at, g.abs()) * some


def likeliest(x, top):
    """Places of the largest values, of equals the lowest first, NaN in front."""
    return torch.sort(x.double().cpu(), dim=-1, descending=True, stable=True).indices[..., :top].to(x.device)
