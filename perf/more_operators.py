"""Dropout and the loss at the end of a model as cases that can be timed on one GPU: dropout by a
counter-based generator (by itself, in front of a layer norm's sum, and of attention probabilities), log
probabilities of given tokens with entropy and the likeliest alternatives, and the cross entropy with its
gradient.  A case is a dict of plain values; `prepare` makes what a program has in hand before the call,
`run` makes one pass: with ``own`` the calls a user makes of ``hipress_b200.ops``, without it the formulas
in elementary torch operations in 32 bits.

Which elements a dropout keeps follows from the seed alone.  Elements are counted in their logical order
(attention probabilities [batch, heads, queries, keys] with the keys rounded up to 32), 32 to a word; word
w of a call with the number `site` has 16 random words, the results of Philox4x32 with 7 rounds and the
seed as its key for the counters (w mod 2^32, w div 2^32, site, 0 .. 3).  Bit i of the j-th is bit j of a
number of 16 bits for element 32 w + i, which is kept where that number is at least 2^16 - t, with t =
(1 - p) 2^16, rounded, and then multiplied by 2^16 / t.
"""
import math

import torch

own = False
DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORED = -100


def listed():
    return [
        # one short sentence through BERT-base, in training: launches decide
        {"name": "dropout 1 sentence", "op": "dropout", "rows": 128, "cols": 768, "type": "bf16", "p": 0.1,
         "residual": False, "site": 3},
        # activations of a wide model in 32 bits, odd sizes everywhere, the half of them dropped, on a residual branch
        {"name": "dropout wide ragged", "op": "dropout", "rows": 8191, "cols": 4999, "type": "fp32", "p": 0.5,
         "residual": True, "site": 1},
        # BERT-large's step, 32 sequences of 128 tokens: what follows every attention and feed-forward layer
        {"name": "norm bert_large", "op": "norm", "rows": 4096, "cols": 1024, "type": "bf16", "weights": "fp32",
         "p": 0.1, "site": 7},
        # many tokens of a model whose width is odd, half precision
        {"name": "norm 32k tokens ragged", "op": "norm", "rows": 32767, "cols": 1021, "type": "fp16",
         "weights": "fp16", "p": 0.3, "site": 0},
        # the decoder of the base Transformer, two short sentences
        {"name": "attention 2 sentences", "op": "attention", "batch": 2, "sq": 33, "sk": 33, "heads": 8,
         "kv_heads": 8, "dim": 64, "type": "fp16", "causal": True, "padding": False, "p": 0.1, "site": 2},
        # BERT-large's step: 32 padded sequences of 128 tokens
        {"name": "attention bert_large", "op": "attention", "batch": 32, "sq": 128, "sk": 128, "heads": 16,
         "kv_heads": 16, "dim": 64, "type": "bf16", "causal": False, "padding": True, "p": 0.1, "site": 5},
        # one long document, causal
        {"name": "attention long", "op": "attention", "batch": 1, "sq": 4096, "sk": 4096, "heads": 16,
         "kv_heads": 16, "dim": 64, "type": "bf16", "causal": True, "padding": False, "p": 0.1, "site": 11},
        # one blank of one sentence is filled in, with the alternatives a user is shown
        {"name": "score 1 token", "op": "score", "rows": 1, "vocab": 30522, "type": "bf16", "top": 5,
         "ignored": 0.0, "training": False},
        # the masked positions of BERT-large's step, trained with an entropy bonus: rows that are not aligned
        {"name": "score masked positions", "op": "score", "rows": 617, "vocab": 30522, "type": "bf16", "top": 0,
         "ignored": 0.0, "training": True},
        # a text of many words judged by the LSTM, in 32 bits, with a long list of alternatives
        {"name": "score text", "op": "score", "rows": 4093, "vocab": 33278, "type": "fp32", "top": 20,
         "ignored": 0.1, "training": False},
        # the loss of BERT-large's step
        {"name": "loss masked positions", "op": "loss", "rows": 617, "vocab": 30522, "type": "bf16",
         "ignored": 0.0},
        # the loss of the base Transformer, 64 padded sentences of 128 words
        {"name": "loss transformer", "op": "loss", "rows": 8192, "vocab": 32000, "type": "fp16", "ignored": 0.25},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _p(rng):
    return rng.choice((0.1, 0.1, 0.5, round(rng.uniform(0.01, 0.9), 3)))


def _draw_dropout(rng):
    cols = rng.choice((512, 768, 1024, _log(rng, 1, 12000), _log(rng, 64, 12000)))
    return {"op": "dropout", "rows": _log(rng, 1, max(1, 8191 * 4999 // cols)), "cols": cols,
            "type": rng.choice(("bf16", "bf16", "fp16", "fp32")), "p": _p(rng), "residual": rng.random() < 0.5,
            "site": rng.randrange(100)}


def _draw_norm(rng):
    cols = rng.choice((512, 768, 1024, _log(rng, 16, 12000), _log(rng, 64, 12000)))
    kind = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    return {"op": "norm", "rows": _log(rng, 1, max(1, 8191 * 4999 // cols)), "cols": cols, "type": kind,
            "weights": rng.choice(("fp32", kind)), "p": _p(rng), "site": rng.randrange(100)}


def _draw_attention(rng):
    dim = rng.choice((64, 64, 128, 128, 32, 8 * rng.randint(1, 16)))
    kv_heads, group = rng.choice((1, 2, 4, 8, 12, 16)), rng.choice((1, 1, 1, 2, 4))
    same = rng.random() < 0.6
    while True:
        # the gradient of a softmax over one key is zero, and what is computed of it rounding alone
        sq = _log(rng, 4 if same else 1, 4096)
        sk = sq if same else _log(rng, 4, 4096)
        batch = _log(rng, 1, 64)
        if batch * kv_heads * group * sq * sk * max(dim, 64) <= 16 * 4096 * 4096 * 32:
            break
    return {"op": "attention", "batch": batch, "sq": sq, "sk": sk, "heads": kv_heads * group, "kv_heads": kv_heads,
            "dim": dim, "type": rng.choice(("bf16", "fp16")), "causal": rng.random() < 0.4,
            "padding": rng.random() < 0.4, "p": _p(rng), "site": rng.randrange(100)}


def _draw_score(rng):
    vocab = rng.choice((30522, 32000, 33278, _log(rng, 50, 200000), _log(rng, 1000, 200000)))
    training = rng.random() < 0.4
    return {"op": "score", "rows": _log(rng, 1, max(1, 4093 * 33278 // vocab // (2 if training else 1))),
            "vocab": vocab, "type": rng.choice(("bf16", "bf16", "fp16", "fp32")),
            "top": rng.choice((0, 1, 5, 20, rng.randint(2, 32))), "ignored": rng.choice((0.0, 0.0, 0.2)),
            "training": training}


def _draw_loss(rng):
    vocab = rng.choice((30522, 32000, 33278, _log(rng, 50, 200000), _log(rng, 1000, 200000)))
    return {"op": "loss", "rows": _log(rng, 1, max(1, 8192 * 16000 // vocab)), "vocab": vocab,
            "type": rng.choice(("bf16", "bf16", "fp16", "fp32")), "ignored": rng.choice((0.0, 0.15, 0.4))}


def draw(rng):
    return rng.choice((_draw_dropout, _draw_norm, _draw_attention, _draw_score, _draw_loss))(rng)


# ------------------------------------------------------------------- inputs
class State(dict):
    __getattr__ = dict.__getitem__


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    t = TYPES[case["type"]]

    def rand(*shape, std=1.0, mean=0.0, dtype=t):
        return torch.randn(*shape, device=DEVICE, generator=gen).mul_(std).add_(mean).to(dtype)

    s = State(case)
    if "p" in case:     # the seed of a step: a number on the device, so that a captured step can move it on
        s["seed"] = torch.randint(0, 2 ** 62, (1,), device=DEVICE, generator=gen)
    wanted = ()
    if case["op"] == "dropout":
        n = case["rows"], case["cols"]
        s.update(x=rand(*n), r=rand(*n) if case["residual"] else None, dy=rand(*n, std=0.1))
        wanted = ("x", "r")
    elif case["op"] == "norm":
        n, w = (case["rows"], case["cols"]), TYPES[case["weights"]]
        s.update(x=rand(*n, std=1.5, mean=0.3), r=rand(*n), weight=rand(n[1], std=0.2, mean=1.0, dtype=w),
                 bias=rand(n[1], std=0.1, dtype=w), dy=rand(*n, std=0.1), dz=rand(*n, std=0.1))
        wanted = ("x", "r", "weight", "bias")
    elif case["op"] == "attention":
        b, sq, sk, h, hk, d = (case[a] for a in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
        if sq == sk and h == hk:   # the projection's output: q, k and v side by side
            s.update(zip("qkv", rand(b, sq, 3, h, d).unbind(2)))
        else:
            s.update(q=rand(b, sq, h, d), k=rand(b, sk, hk, d), v=rand(b, sk, hk, d))
        s.update(do=rand(b, sq, h, d, std=0.1), mask=None)
        if case["padding"]:        # every sequence has a length of its own, of at least half the longest
            lengths = torch.randint((sk + 1) // 2, sk + 1, (b, 1), device=DEVICE, generator=gen)
            s["mask"] = torch.arange(sk, device=DEVICE)[None] < lengths
        wanted = ("q", "k", "v")
    else:
        rows, vocab = case["rows"], case["vocab"]
        # a model that has learnt something: the given token stands out, by more or less
        tokens = torch.randint(0, vocab, (rows,), device=DEVICE, generator=gen)
        logits = torch.randn(rows, vocab, device=DEVICE, generator=gen).mul_(2.0)
        logits[torch.arange(rows, device=DEVICE), tokens] += 8 * torch.rand(rows, device=DEVICE, generator=gen)
        if case["ignored"]:
            gone = torch.rand(rows, device=DEVICE, generator=gen) < case["ignored"]
            gone[0] = False
            tokens = torch.where(gone, IGNORED, tokens)
        s.update(logits=logits.to(t), tokens=tokens)
        if case["op"] == "loss":   # fp16 is trained with a scaled loss: gradients would vanish
            s["scale"] = torch.tensor(65536.0 if case["type"] == "fp16" else 1.0, device=DEVICE)
        if case["op"] == "loss" or case["training"]:
            wanted = ("logits",)
        if case["op"] == "score" and case["training"]:
            s.update(dlogp=rand(rows, std=0.1, dtype=torch.float32), dentropy=rand(rows, std=0.02, dtype=torch.float32))
    for name in wanted:
        if s[name] is not None:
            s[name] = s[name].detach().requires_grad_(True)
    return s


# ------------------------------------------------------- the framework's calls
def _own_dropout(s):
    from hipress_b200.ops import dropout
    y = dropout(s.x, s.p, seed=s.seed, site=s.site, residual=s.r)
    if s.r is None:
        dx, = torch.autograd.grad(y, (s.x,), s.dy)
        return {"y": y, "dx": dx}
    dx, dr = torch.autograd.grad(y, (s.x, s.r), s.dy)
    return {"y": y, "dx": dx, "dr": dr}


def _own_norm(s):
    from hipress_b200.ops import layer_norm
    y, z = layer_norm(s.x, s.weight, s.bias, residual=s.r, dropout=s.p, seed=s.seed, site=s.site)
    dx, dr, dw, db = torch.autograd.grad((y, z), (s.x, s.r, s.weight, s.bias), (s.dy, s.dz))
    return {"y": y, "z": z, "dx": dx, "dr": dr, "dw": dw, "db": db}


def _own_attention(s):
    from hipress_b200.ops import attention
    out, lse = attention(s.q, s.k, s.v, causal=s.causal, key_mask=s.mask, return_lse=True, dropout=s.p, seed=s.seed,
                         site=s.site)
    dq, dk, dv = torch.autograd.grad(out, (s.q, s.k, s.v), s.do)
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _own_score(s):
    from hipress_b200.ops import token_log_probs
    got = token_log_probs(s.logits, s.tokens, top=s.top, ignore_index=IGNORED)
    out = {"logp": got.log_probs, "entropy": got.entropy}
    if s.top:
        out.update(top_logp=got.top_log_probs, top=got.top_tokens)
    if s.training:
        out["dlogits"], = torch.autograd.grad((got.log_probs, got.entropy), (s.logits,), (s.dlogp, s.dentropy))
    return out


def _own_loss(s):
    from hipress_b200.ops import cross_entropy
    loss = cross_entropy(s.logits, s.tokens, ignore_index=IGNORED)
    dlogits, = torch.autograd.grad(loss, (s.logits,), s.scale)
    return {"loss": loss, "dlogits": dlogits}


# --------------------------------------------------------------- plain forms
def _philox(c, key):
    """Philox4x32 with 7 rounds: four words for each counter (c: four tensors or numbers, key: two tensors)."""
    mask = 0xFFFFFFFF
    x0, x1, x2, x3 = c
    k0, k1 = key
    for _ in range(7):
        p0, p1 = x0 * 0xD2511F53, x2 * 0xCD9E8D57    # 64 bits; the sign bit is one of them
        x0, x1, x2, x3 = (p1 >> 32 & mask) ^ x1 ^ k0, p1 & mask, (p0 >> 32 & mask) ^ x3 ^ k1, p0 & mask
        k0, k1 = k0 + 0x9E3779B9 & mask, k1 + 0xBB67AE85 & mask
    return x0, x1, x2, x3


def _kept(first, words, s):
    """Whether each element of the words from the given one on is kept."""
    t = round((1 - s.p) * 65536)
    w = torch.arange(first, first + words, device=s.seed.device)
    key = s.seed & 0xFFFFFFFF, s.seed >> 32 & 0xFFFFFFFF
    keep = torch.zeros_like(w)
    for call in range(4):
        for j, r in enumerate(_philox((w & 0xFFFFFFFF, w >> 32, torch.full_like(w, s.site), torch.full_like(w, call)), key)):
            keep = keep | r if t >> (4 * call + j) & 1 else keep & r
    bits = torch.arange(32, device=w.device, dtype=torch.int32)
    return (keep.to(torch.int32)[:, None] >> bits & 1).bool().flatten(), 65536 / t


def _plain_dropout(s):
    t, n = s.x.dtype, s.rows * s.cols
    keep, up = _kept(0, (n + 31) // 32, s)
    keep = keep[:n].view(s.rows, s.cols)
    y = torch.where(keep, s.x.float() * up, 0.0)
    out = {"y": (y if s.r is None else y + s.r.float()).to(t), "dx": torch.where(keep, s.dy.float() * up, 0.0).to(t)}
    if s.r is not None:
        out["dr"] = s.dy.clone()
    return out


def _plain_norm(s):
    t, w, b, n = s.x.dtype, s.weight.float(), s.bias.float(), s.rows * s.cols
    keep, up = _kept(0, (n + 31) // 32, s)
    keep = keep[:n].view(s.rows, s.cols)
    zt = (torch.where(keep, s.x.float() * up, 0.0) + s.r.float()).to(t)   # the sum is an output, and what is normalised
    z = zt.float()
    mean = z.mean(1, keepdim=True)
    c = z - mean
    rstd = (c.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    h = c * rstd
    dy = s.dy.float()
    g = dy * w
    dr = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True)) + s.dz.float()
    return {"y": (h * w + b).to(t), "z": zt, "dx": torch.where(keep, dr * up, 0.0).to(t), "dr": dr.to(t),
            "dw": (dy * h).sum(0).to(s.weight.dtype), "db": dy.sum(0).to(s.bias.dtype)}


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
    per_row = (sk + 31) // 32
    rows = b * hk * group * sq
    keep, up = _kept(0, rows * per_row, s)
    keep = keep.view(rows, 32 * per_row)[:, :sk].reshape(p.shape)
    dropped = torch.where(keep, p * up, 0.0)
    o = dropped @ v
    do = heads(s.do)
    dv = back(dropped.transpose(2, 3) @ do, sk)
    delta = (do * o).sum(-1, keepdim=True)
    ds = torch.where(keep, (do @ v.transpose(2, 3)).mul_(up), 0.0).sub_(delta).mul_(p).mul_(scale)
    return {"out": back(o, sq), "lse": lse, "dq": back(ds @ k, sq), "dk": back(ds.transpose(2, 3) @ q, sk), "dv": dv}


def _log_probs(s):
    x = s.logits.float()
    lse = x.amax(1, keepdim=True)
    lse = lse + (x - lse).exp().sum(1, keepdim=True).log()
    return x - lse


def _plain_score(s):
    t, lp = s.logits.dtype, _log_probs(s)
    there = s.tokens != IGNORED
    at = torch.where(there, s.tokens, 0)[:, None]
    p = lp.exp()
    entropy = -(p * lp).sum(1)
    out = {"logp": torch.where(there, lp.gather(1, at)[:, 0], 0.0), "entropy": entropy}
    if s.top:
        order = torch.sort(s.logits, dim=1, descending=True, stable=True).indices[:, :s.top]   # ties: the lowest first
        out.update(top_logp=lp.gather(1, order), top=order)
    if s.training:
        g = torch.where(there, s.dlogp, 0.0)[:, None]
        d = -p * (g + s.dentropy[:, None] * (lp + entropy[:, None]))
        out["dlogits"] = d.scatter_add_(1, at, g).to(t)
    return out


def _plain_loss(s):
    t, lp = s.logits.dtype, _log_probs(s)
    there = s.tokens != IGNORED
    at = torch.where(there, s.tokens, 0)[:, None]
    n = there.sum()
    loss = -torch.where(there, lp.gather(1, at)[:, 0], 0.0).sum() / n
    g = (there.float() / n * s.scale)[:, None]
    return {"loss": loss, "dlogits": (lp.exp() * g).scatter_add_(1, at, -g).to(t)}


def run(state):
    forms = {"dropout": (_plain_dropout, _own_dropout), "norm": (_plain_norm, _own_norm),
             "attention": (_plain_attention, _own_attention), "score": (_plain_score, _own_score),
             "loss": (_plain_loss, _own_loss)}[state["op"]]
    if own:
        return forms[1](state)
    with torch.no_grad():
        return forms[0](state)


# ------------------------------------------------------------------ the work
def work(case):
    e = 4 if case["type"] == "fp32" else 2
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        # forward x (r) -> y, backward dy -> dx
        return {"bytes": n * e * (5 if case["residual"] else 4), "flops": 3 * n}
    if case["op"] == "norm":
        n, w = case["rows"] * case["cols"], 4 if case["weights"] == "fp32" else 2
        # forward x r -> y z, backward z dy dz -> dx dr; weight, bias and their gradients
        return {"bytes": n * e * 9 + 5 * case["cols"] * w, "flops": 20 * n}
    if case["op"] == "attention":
        b, sq, sk, h, hk, d = (case[a] for a in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
        nq, nk = b * sq * h, b * sk * hk
        pairs = sq * sk
        if case["causal"]:
            short = min(sq, sk)   # rows that see something
            pairs = short * (short + 1) // 2 + short * max(sk - sq, 0)
        return {"bytes": e * d * (4 * nq + 4 * nk) + 4 * nq, "flops": 14 * d * pairs * b * h}
    n = case["rows"] * case["vocab"]
    training = case["op"] == "loss" or case["training"]
    # forward logits, backward logits -> their gradient; tokens and results of each row
    return {"bytes": n * e * (3 if training else 1) + case["rows"] * (16 + 12 * case.get("top", 0)),
            "flops": n * (8 if training else 4)}


# ------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f = {k: v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    with torch.no_grad():
        return {"dropout": _exact_dropout, "norm": _exact_norm, "attention": _exact_attention, "score": _exact_score,
                "loss": _exact_loss}[case["op"]](f, s)


def _numbers(first, words, s):
    """The elements' numbers of 16 bits; the 64-bit products of the generator in parts of 16 bits."""
    def times(m, x):      # upper and lower word of m x
        lo, hi = m * (x & 0xFFFF), m * (x >> 16)     # 48 bits each
        total = lo + ((hi & 0xFFFF) << 16)
        return (hi >> 16) + (total >> 32), total & 0xFFFFFFFF

    seed = int(s["seed"])
    w = first + torch.arange(words, device=DEVICE)
    u = torch.zeros(words, 32, dtype=torch.int32, device=DEVICE)
    places = torch.arange(32, device=DEVICE)
    for call in range(4):
        x = [w % 2 ** 32, w // 2 ** 32, torch.zeros_like(w) + s["site"], torch.zeros_like(w) + call]
        for i in range(7):
            h0, l0 = times(0xD2511F53, x[0])
            h1, l1 = times(0xCD9E8D57, x[2])
            x = [h1 ^ x[1] ^ (seed + i * 0x9E3779B9) % 2 ** 32, l1, h0 ^ x[3] ^ ((seed >> 32) + i * 0xBB67AE85) % 2 ** 32, l0]
        for j, r in enumerate(x):
            u += ((r[:, None] >> places) % 2 << (4 * call + j)).to(torch.int32)
    return u


def _factors(s, rows, cols, per_row=None, first=0):
    """What each element is multiplied by: zero, or the inverse of the share that is kept."""
    t = round((1 - s["p"]) * 65536)
    n = rows * cols if per_row is None else rows * per_row * 32
    parts = []
    for at in range(0, (n + 31) // 32, 1 << 22):      # a part at a time: a word takes 400 bytes on the way
        u = _numbers(first + at, min(1 << 22, (n + 31) // 32 - at), s)
        parts.append((u >= 65536 - t).flatten())
    keep = torch.cat(parts)[:n]
    keep = keep.view(rows, cols) if per_row is None else keep.view(rows, per_row * 32)[:, :cols]
    return keep.double() * (65536 / t)


def _exact_dropout(f, s):
    m = _factors(s, s.rows, s.cols)
    out = {"y": f["x"] * m, "dx": f["dy"] * m}
    if s.r is not None:
        out.update(y=out["y"] + f["r"], dr=f["dy"])
    return out


def _exact_norm(f, s):
    m = _factors(s, s.rows, s.cols)
    sum_ = f["x"] * m + f["r"]
    z = sum_.to(s.x.dtype).double()
    var, mean = torch.var_mean(z, 1, unbiased=False, keepdim=True)
    sigma = torch.sqrt(var + 1e-5)
    h = (z - mean) / sigma
    # the Jacobian's rows, from d(h)/d(z) = (1 - 1/C - h h^T / C) / sigma
    u = f["dy"] * f["weight"]
    c = z.shape[1]
    dr = (u - (u.sum(1, keepdim=True) + h * torch.einsum("rc,rc->r", u, h)[:, None]) / c) / sigma + f["dz"]
    return {"y": torch.addcmul(f["bias"], h, f["weight"]), "z": sum_, "dx": dr * m, "dr": dr,
            "dw": torch.einsum("rc,rc->c", f["dy"], h), "db": f["dy"].sum(0)}


def _exact_attention(f, s):
    b, sq, sk, h, hk, d = (s[a] for a in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
    q, k, v, do = f["q"], f["k"], f["v"], f["do"]
    like = {"out": q, "dq": q, "dk": k, "dv": v}
    out = {name: torch.zeros(x.shape, dtype=torch.float64, device=q.device) for name, x in like.items()}
    out["lse"] = torch.empty(b, h, sq, dtype=torch.float64, device=q.device)
    seen = torch.ones(sq, sk, dtype=torch.bool, device=q.device)
    if s.causal:
        seen = seen.tril(sk - sq)
    per_row = -(-sk // 32)
    for i in range(b):
        see = seen if s.mask is None else seen & s.mask[i][None]
        factors = _factors(s, h * sq, sk, per_row, i * h * sq * per_row).view(h, sq, sk)
        for j in range(h):       # one query head at a time: its matrices of sq x sk fit easily
            kj = j // (h // hk)
            x = torch.where(see, q[i, :, j] @ k[i, :, kj].t() / math.sqrt(d), -math.inf)
            lse = torch.logsumexp(x, 1)
            p = torch.exp(x - torch.where(lse == -math.inf, 0.0, lse)[:, None])
            m = factors[j]
            pm = p * m
            g = do[i, :, j]
            out["out"][i, :, j], out["lse"][i, j] = pm @ v[i, :, kj], lse
            out["dv"][i, :, kj] += pm.t() @ g
            dp = (g @ v[i, :, kj].t()) * m
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(d)
            out["dq"][i, :, j] = ds @ k[i, :, kj]
            out["dk"][i, :, kj] += ds.t() @ q[i, :, j]
    return out


def _exact_rows(f, s):
    """In parts of the rows: log probabilities, and which rows have a token."""
    for at in range(0, s.rows, 1024):
        x = s.logits[at:at + 1024].detach().double()
        yield slice(at, at + 1024), x - torch.logsumexp(x, 1, keepdim=True)


def _exact_score(f, s):
    rows, top = s.rows, s.top
    out = {"logp": torch.zeros(rows, dtype=torch.float64, device=DEVICE), "entropy": torch.empty(rows, dtype=torch.float64, device=DEVICE)}
    if top:
        out.update(top_logp=torch.empty(rows, top, dtype=torch.float64, device=DEVICE),
                   top=torch.empty(rows, top, dtype=torch.int64, device=DEVICE))
    if s.training:
        out["dlogits"] = torch.empty(rows, s.vocab, dtype=torch.float64, device=DEVICE)
    for part, lp in _exact_rows(f, s):
        tokens = s.tokens[part]
        here = (tokens != IGNORED).nonzero()[:, 0]
        index = torch.arange(part.start, part.start + lp.shape[0], device=DEVICE)
        out["logp"][index[here]] = lp[here, tokens[here]]
        p = torch.exp(lp)
        out["entropy"][part] = h = -torch.einsum("rv,rv->r", p, lp)
        if top:    # the largest again and again, the first of equals
            left = s.logits[part].detach().double()
            for i in range(top):
                best = left.amax(1, keepdim=True)
                at = torch.where(left == best, torch.arange(s.vocab, device=DEVICE), s.vocab).amin(1, keepdim=True)
                out["top"][part, i], out["top_logp"][part, i] = at[:, 0], lp.gather(1, at)[:, 0]
                left.scatter_(1, at, -math.inf)
        if s.training:
            # d logp_y / d x = 1_y - p,  d H / d x = -p (logp + H)
            g = -p * (lp + h[:, None]) * f["dentropy"][part][:, None]
            ones = torch.zeros_like(p)
            ones[here, tokens[here]] = 1.0
            g[here] += (ones[here] - p[here]) * f["dlogp"][part][here][:, None]
            out["dlogits"][part] = g
    return out


def _exact_loss(f, s):
    n = int((s.tokens != IGNORED).sum())
    total = torch.zeros((), dtype=torch.float64, device=DEVICE)
    d = torch.zeros(s.rows, s.vocab, dtype=torch.float64, device=DEVICE)
    for part, lp in _exact_rows(f, s):
        tokens = s.tokens[part]
        here = (tokens != IGNORED).nonzero()[:, 0]
        total -= lp[here, tokens[here]].sum()
        g = torch.exp(lp)
        g[here, tokens[here]] -= 1.0
        d[part][here] = g[here] / n * float(s.scale)
    return {"loss": total / n, "dlogits": d}
