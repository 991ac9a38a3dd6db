"""The layer operators as cases that can be timed on one GPU: layer norm, the matrix product
with its epilogue (``linear``) and attention, forward or as a training step (forward and
gradients).  A case is a dict of plain values; `prepare` makes what a program has in hand
before the call, `run` makes one pass: with ``own`` the calls a user makes of
``hipress_b200.ops``, without it the formulas in elementary torch operations in 32 bits.
"""
import math

import torch

own = False
DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one short sentence through BERT-base: a few microseconds of GPU work, launches decide
        {"name": "norm 1 sentence", "op": "norm", "rows": 128, "cols": 768, "type": "bf16", "weights": "fp32",
         "residual": False},
        # BERT-large's step, 32 sequences of 128 tokens, under autocast: fp32 weights, the residual sum in front
        {"name": "norm bert_large residual", "op": "norm", "rows": 4096, "cols": 1024, "type": "bf16",
         "weights": "fp32", "residual": True},
        # a wide model in half precision, odd sizes everywhere
        {"name": "norm wide ragged", "op": "norm", "rows": 8191, "cols": 4999, "type": "fp16", "weights": "fp16",
         "residual": True},
        # 128 sequences of the longest kind (512 tokens): larger than the L2 cache
        {"name": "norm 64k tokens", "op": "norm", "rows": 65536, "cols": 1024, "type": "bf16", "weights": "fp32",
         "residual": False},
        # the feed-forward layer of the base Transformer (512 -> 2048) for one short sentence
        {"name": "linear few rows", "op": "linear", "m": 33, "k": 512, "n": 2048, "type": "fp16", "weights": "fp16",
         "activation": "relu", "residual": False, "training": True},
        # BERT-large's step: feed-forward up (with GELU) and down (with the residual, fp32 weights and their gradient)
        {"name": "linear bert_large up", "op": "linear", "m": 4096, "k": 1024, "n": 4096, "type": "bf16",
         "weights": "bf16", "activation": "gelu", "residual": False, "training": True},
        {"name": "linear bert_large down", "op": "linear", "m": 4096, "k": 4096, "n": 1024, "type": "bf16",
         "weights": "fp32", "activation": None, "residual": True, "training": True},
        # the vocabulary projection of the masked positions: rows of 30522 values, which are not aligned
        {"name": "linear vocabulary", "op": "linear", "m": 617, "k": 1024, "n": 30522, "type": "bf16",
         "weights": "fp32", "activation": None, "residual": False, "training": True},
        # the decoder of the base Transformer, two short sentences
        {"name": "attention 2 sentences", "op": "attention", "batch": 2, "sq": 33, "sk": 33, "heads": 8,
         "kv_heads": 8, "dim": 64, "type": "fp16", "causal": True, "padding": False, "training": True},
        # BERT-large's step: 32 padded sequences of 128 tokens, q, k and v as one projection leaves them
        {"name": "attention bert_large", "op": "attention", "batch": 32, "sq": 128, "sk": 128, "heads": 16,
         "kv_heads": 16, "dim": 64, "type": "bf16", "causal": False, "padding": True, "training": True},
        # cross attention over a ragged memory, shared key heads, wide heads
        {"name": "attention cross ragged", "op": "attention", "batch": 8, "sq": 517, "sk": 1999, "heads": 16,
         "kv_heads": 4, "dim": 128, "type": "fp16", "causal": False, "padding": True, "training": True},
        # one long document, causal
        {"name": "attention long", "op": "attention", "batch": 1, "sq": 8192, "sk": 8192, "heads": 16,
         "kv_heads": 16, "dim": 64, "type": "bf16", "causal": True, "padding": False, "training": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_norm(rng):
    cols = rng.choice((512, 768, 1024, _log(rng, 16, 12000), _log(rng, 64, 12000)))
    kind = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    return {"op": "norm", "rows": _log(rng, 1, max(1, min(65536, (65536 * 1024) // cols))), "cols": cols,
            "type": kind, "weights": rng.choice(("fp32", kind)), "residual": rng.random() < 0.5}


def _draw_linear(rng):
    while True:
        m = _log(rng, 1, 32768)
        n, k = ((rng.choice((512, 768, 1024, 2048, 4096)) if rng.random() < 0.4 else _log(rng, 8, 8192)) for _ in range(2))
        training = rng.random() < 0.75
        if m * n * k * (3 if training else 1) <= 3 * 617 * 1024 * 30522:
            break
    kind = rng.choice(("bf16", "bf16", "fp16"))
    activation = rng.choice((None, "relu", "gelu", "gelu_tanh"))
    # fp32 weights: their gradient comes in 32 bits
    return {"op": "linear", "m": m, "k": k, "n": n, "type": kind,
            "weights": kind if activation else rng.choice((kind, "fp32")), "activation": activation,
            "residual": rng.random() < 0.4, "training": training}


def _draw_attention(rng):
    dim = rng.choice((64, 64, 128, 128, 32, 8 * rng.randint(1, 16)))
    kv_heads, group = rng.choice((1, 2, 4, 8, 12, 16)), rng.choice((1, 1, 1, 2, 4))
    same = rng.random() < 0.6
    training = rng.random() < 0.7
    # the gradient of a softmax over one key is zero, and what is computed of it rounding alone
    least = 4 if training else 1
    while True:
        sq = _log(rng, least if same else 1, 8192)
        sk = sq if same else _log(rng, least, 8192)
        batch = _log(rng, 1, 64)
        if batch * kv_heads * group * sq * sk * max(dim, 64) <= 16 * 8192 * 8192 * 32:
            break
    return {"op": "attention", "batch": batch, "sq": sq, "sk": sk, "heads": kv_heads * group, "kv_heads": kv_heads,
            "dim": dim, "type": rng.choice(("bf16", "fp16")), "causal": rng.random() < 0.4,
            "padding": rng.random() < 0.4, "training": training}


def draw(rng):
    return rng.choice((_draw_norm, _draw_linear, _draw_attention))(rng)


# ------------------------------------------------------------------- inputs
class State(dict):
    __getattr__ = dict.__getitem__


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    t = TYPES[case["type"]]

    def rand(*shape, std=1.0, mean=0.0, dtype=t):
        return torch.randn(*shape, device=DEVICE, generator=gen).mul_(std).add_(mean).to(dtype)

    s = State(case)
    if case["op"] == "norm":
        rows, cols, w = case["rows"], case["cols"], TYPES[case["weights"]]
        s.update(x=rand(rows, cols, std=1.5, mean=0.3), weight=rand(cols, std=0.2, mean=1.0, dtype=w),
                 bias=rand(cols, std=0.1, dtype=w), r=rand(rows, cols) if case["residual"] else None,
                 dy=rand(rows, cols, std=0.1), dz=rand(rows, cols, std=0.1) if case["residual"] else None)
        wanted = ("x", "weight", "bias", "r")
    elif case["op"] == "linear":
        m, n, k, w = case["m"], case["n"], case["k"], TYPES[case["weights"]]
        s.update(x=rand(m, k), weight=rand(n, k, std=k ** -0.5, dtype=w), bias=rand(n, std=0.1, dtype=w),
                 r=rand(m, n) if case["residual"] else None, dy=rand(m, n, std=0.1) if case["training"] else None)
        wanted = ("x", "weight", "bias", "r") if case["training"] else ()
    else:
        b, sq, sk, h, hk, d = (case[a] for a in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
        if sq == sk and h == hk:   # the projection's output: q, k and v side by side
            qkv = rand(b, sq, 3, h, d)
            s.update(zip("qkv", qkv.unbind(2)))
        else:
            s.update(q=rand(b, sq, h, d), k=rand(b, sk, hk, d), v=rand(b, sk, hk, d))
        s.update(do=rand(b, sq, h, d, std=0.1) if case["training"] else None, mask=None)
        if case["padding"]:        # every sequence has a length of its own, of at least half the longest
            lengths = torch.randint((sk + 1) // 2, sk + 1, (b, 1), device=DEVICE, generator=gen)
            s["mask"] = torch.arange(sk, device=DEVICE)[None] < lengths
        wanted = ("q", "k", "v") if case["training"] else ()
    for name in wanted:
        if s[name] is not None:
            s[name] = s[name].detach().requires_grad_(True)
    return s


# ------------------------------------------------------- the framework's calls
def _own_norm(s):
    from hipress_b200.ops import layer_norm
    if s.r is None:
        y = layer_norm(s.x, s.weight, s.bias)
        dx, dw, db = torch.autograd.grad(y, (s.x, s.weight, s.bias), s.dy)
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    y, z = layer_norm(s.x, s.weight, s.bias, residual=s.r)
    dx, dw, db, dr = torch.autograd.grad((y, z), (s.x, s.weight, s.bias, s.r), (s.dy, s.dz))
    return {"y": y, "z": z, "dx": dx, "dw": dw, "db": db, "dr": dr}


def _own_linear(s):
    from hipress_b200.ops import linear
    y = linear(s.x, s.weight, s.bias, activation=s.activation, residual=s.r)
    if not s.training:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (s.x, s.weight, s.bias), s.dy)
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def _own_attention(s):
    from hipress_b200.ops import attention
    out, lse = attention(s.q, s.k, s.v, causal=s.causal, key_mask=s.mask, return_lse=True)
    if not s.training:
        return {"out": out, "lse": lse}
    dq, dk, dv = torch.autograd.grad(out, (s.q, s.k, s.v), s.do)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


# --------------------------------------------------------------- plain forms
def _plain_norm(s):
    t, w, b = s.x.dtype, s.weight.float(), s.bias.float()
    z = s.x.float()
    if s.r is not None:
        zt = (z + s.r.float()).to(t)   # the sum is an output, and what is normalised
        z = zt.float()
    mean = z.mean(1, keepdim=True)
    c = z - mean
    rstd = (c.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    h = c * rstd
    y = h * w + b
    dy = s.dy.float()
    g = dy * w
    dz = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    out = {"y": y.to(t), "dw": (dy * h).sum(0).to(s.weight.dtype), "db": dy.sum(0).to(s.bias.dtype)}
    if s.r is not None:
        dz = (dz + s.dz.float()).to(t)
        return {**out, "z": zt, "dx": dz, "dr": dz}
    return {**out, "dx": dz.to(t)}


def _act(p, kind):
    """The activation and its derivative."""
    if kind is None:
        return p, None
    if kind == "relu":
        return p.clamp(min=0), (p > 0).to(p.dtype)
    if kind == "gelu":
        cdf = 0.5 * (1 + torch.erf(p * math.sqrt(0.5)))
        return p * cdf, cdf + p * torch.exp(-0.5 * p * p) / math.sqrt(2 * math.pi)
    c, a = math.sqrt(2 / math.pi), 0.044715
    th = torch.tanh(c * (p + a * p * p * p))
    return 0.5 * p * (1 + th), 0.5 * (1 + th) + 0.5 * p * (1 - th * th) * c * (1 + 3 * a * p * p)


def _plain_linear(s):
    t, x, w = s.x.dtype, s.x.float(), s.weight.float()
    y, slope = _act(x @ w.t() + s.bias.float(), s.activation)
    if s.r is not None:
        y = y + s.r.float()
    if not s.training:
        return {"y": y.to(t)}
    g = s.dy.float()
    if slope is not None:
        g = g * slope
    return {"y": y.to(t), "dx": (g @ w).to(t), "dw": (g.t() @ x).to(s.weight.dtype), "db": g.sum(0).to(s.bias.dtype)}


def _plain_attention(s):
    t, scale, group = s.q.dtype, s.dim ** -0.5, s.heads // s.kv_heads
    b, sq, sk, hk, d = s.batch, s.sq, s.sk, s.kv_heads, s.dim

    def heads(x):   # [batch, length, heads, d] -> [batch, key heads, group * length, d]
        return x.float().transpose(1, 2).reshape(b, hk, -1, d)

    def back(x, length):
        return x.reshape(b, -1, length, d).transpose(1, 2).to(t).contiguous()

    q, k, v = heads(s.q), heads(s.k), heads(s.v)
    sc = (q @ k.transpose(2, 3)).mul_(scale).view(b, hk, group, sq, sk)
    hidden = None
    if s.causal:
        i, j = torch.arange(sq, device=q.device), torch.arange(sk, device=q.device)
        hidden = (j[None] > i[:, None] + (sk - sq))[None, None, None]
    if s.mask is not None:
        pad = ~s.mask[:, None, None, None]
        hidden = pad if hidden is None else hidden | pad
    if hidden is not None:
        sc = sc.masked_fill_(hidden, -math.inf)
    top = sc.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = sc.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (top + total.log()).reshape(b, -1, sq)
    p = p.div_(torch.where(total == 0, 1.0, total)).view(b, hk, group * sq, sk)
    o = p @ v
    out = {"out": back(o, sq), "lse": lse}
    if not s.training:
        return out
    do = heads(s.do)
    out["dv"] = back(p.transpose(2, 3) @ do, sk)
    delta = (do * o).sum(-1, keepdim=True)
    ds = (do @ v.transpose(2, 3)).sub_(delta).mul_(p).mul_(scale)
    out["dq"] = back(ds @ k, sq)
    out["dk"] = back(ds.transpose(2, 3) @ q, sk)
    return out


def run(state):
    forms = {"norm": (_plain_norm, _own_norm), "linear": (_plain_linear, _own_linear),
             "attention": (_plain_attention, _own_attention)}[state["op"]]
    if own:
        return forms[1](state)
    with torch.no_grad():
        return forms[0](state)


# ------------------------------------------------------------------ the work
def work(case):
    e, w = (4 if case.get(a) == "fp32" else 2 for a in ("type", "weights"))
    if case["op"] == "norm":
        n, c = case["rows"] * case["cols"], case["cols"]
        # forward x (r) -> y (z), backward z dy (dz) -> dx; weight, bias and their gradients
        return {"bytes": n * e * (8 if case["residual"] else 5) + 5 * c * w, "flops": 18 * n}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        forward = e * (m * k + m * n * (2 if case["residual"] else 1)) + w * (n * k + n)
        if not case["training"]:
            return {"bytes": forward, "flops": 2 * m * n * k}
        return {"bytes": forward + e * (m * n + m * k) + w * (n * k + n), "flops": 6 * m * n * k}
    b, sq, sk, h, hk, d = (case[a] for a in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
    nq, nk = b * sq * h, b * sk * hk
    pairs = sq * sk
    if case["causal"]:
        short = min(sq, sk)   # rows that see something
        pairs = short * (short + 1) // 2 + short * max(sk - sq, 0)
    pairs *= b * h
    if not case["training"]:
        return {"bytes": e * d * 2 * (nq + nk) + 4 * nq, "flops": 4 * d * pairs}
    return {"bytes": e * d * (4 * nq + 4 * nk) + 4 * nq, "flops": 14 * d * pairs}


# ------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f = {k: v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    with torch.no_grad():
        return {"norm": _exact_norm, "linear": _exact_linear, "attention": _exact_attention}[case["op"]](f, s)


def _exact_norm(f, s):
    z = f["x"]
    if f["r"] is not None:
        z = (f["x"] + f["r"]).to(s.x.dtype).double()
    var, mean = torch.var_mean(z, 1, unbiased=False, keepdim=True)
    sigma = torch.sqrt(var + 1e-5)
    h = (z - mean) / sigma
    # the Jacobian's rows, from d(h)/d(z) = (1 - 1/C - h h^T / C) / sigma
    u = f["dy"] * f["weight"]
    c = z.shape[1]
    dz = (u - (u.sum(1, keepdim=True) + h * torch.einsum("rc,rc->r", u, h)[:, None]) / c) / sigma
    out = {"y": torch.addcmul(f["bias"], h, f["weight"]), "dw": torch.einsum("rc,rc->c", f["dy"], h),
           "db": f["dy"].sum(0), "dx": dz}
    if f["r"] is not None:
        dz = dz + f["dz"]
        out.update(z=f["x"] + f["r"], dx=dz, dr=dz)
    return out


def _exact_linear(f, s):
    p = torch.addmm(f["bias"], f["x"], f["weight"].t())
    kind = f["activation"]
    if kind == "relu":
        y, slope = torch.where(p > 0, p, 0.0), torch.where(p > 0, 1.0, 0.0).double()
    elif kind == "gelu":
        tail = torch.special.erfc(-p / math.sqrt(2)) / 2
        y, slope = p * tail, tail + p * torch.exp(-p * p / 2) / math.sqrt(2 * math.pi)
    elif kind == "gelu_tanh":
        u = math.sqrt(2 / math.pi) * (p + 0.044715 * p ** 3)
        gate = torch.sigmoid(2 * u)
        y = p * gate
        slope = gate + p * gate * (1 - gate) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * p * p)
    else:
        y, slope = p, None
    if f["r"] is not None:
        y = y + f["r"]
    if not f["training"]:
        return {"y": y}
    g = f["dy"] if slope is None else f["dy"] * slope
    return {"y": y, "dx": g @ f["weight"], "dw": g.t() @ f["x"], "db": g.sum(0)}


def _exact_attention(f, s):
    b, sq, sk, h, hk, d = (s[a] for a in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
    q, k, v, do = f["q"], f["k"], f["v"], f["do"]
    like = {"out": q, "dq": q, "dk": k, "dv": v}
    out = {name: torch.zeros(x.shape, dtype=torch.float64, device=q.device) for name, x in like.items()}
    out["lse"] = torch.empty(b, h, sq, dtype=torch.float64, device=q.device)
    seen = torch.ones(sq, sk, dtype=torch.bool, device=q.device)
    if s.causal:
        seen = seen.tril(sk - sq)
    for i in range(b):
        see = seen if s.mask is None else seen & s.mask[i][None]
        for j in range(h):       # one query head at a time: its matrices of sq x sk fit easily
            kj = j // (h // hk)
            x = torch.where(see, q[i, :, j] @ k[i, :, kj].t() / math.sqrt(d), -math.inf)
            lse = torch.logsumexp(x, 1)
            p = torch.exp(x - torch.where(lse == -math.inf, 0.0, lse)[:, None])
            out["lse"][i, j], out["out"][i, :, j] = lse, p @ v[i, :, kj]
            if s.training:
                g = do[i, :, j]
                out["dv"][i, :, kj] += p.t() @ g
                dp = g @ v[i, :, kj].t()
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(d)
                out["dq"][i, :, j] = ds @ k[i, :, kj]
                out["dk"][i, :, kj] += ds.t() @ q[i, :, j]
    return out if s.training else {"out": out["out"], "lse": out["lse"]}
