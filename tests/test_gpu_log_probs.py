"""Log probabilities and the cross entropy: their kernels against the formulas in 64 bits."""
import math

import pytest
import torch

from _dropout import likeliest, log_probs64, log_probs64_gradient
from _layers import U
from hipress_b200.ops import cross_entropy, token_log_probs

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def steps(vocab):
    """Roundings of a sum over the vocabulary, each 2^-24 of it: a thread's additions one after the other, the
    joins, 2^z (2^-22) and the rounding of z."""
    return 128 + vocab / 64


def check(x, t, top=0, ignored=-100, gradients=True):
    vocab, dtype = x.shape[-1], x.dtype
    leaf = x.detach().requires_grad_(True)
    p = token_log_probs(leaf, t, top=top, ignore_index=ignored)
    lp, want, entropy = log_probs64(x, t, ignored)
    tol = steps(vocab) * 2 ** -24
    assert p.log_probs.dtype == p.entropy.dtype == FP32
    near = lambda a, b, bound: bool(((a.double() - b).abs() <= bound)[torch.isfinite(b)].all()) and \
        torch.equal(a.double()[~torch.isfinite(b)], b[~torch.isfinite(b)])  # noqa: E731
    assert near(p.log_probs, want, tol + 2 ** -22 * want.abs())
    assert near(p.entropy, entropy, tol * (2 + 2 * math.log(vocab + 1)))
    if top:
        best = likeliest(x, top)
        assert torch.equal(p.top_tokens, best)
        values = lp.gather(-1, best)
        assert near(p.top_log_probs, values, tol + 2 ** -22 * values.abs())
    # without the others' results the same
    assert torch.equal(token_log_probs(x, t, entropy=False, ignore_index=ignored).log_probs, p.log_probs)
    if gradients:
        g, h = (torch.randn(t.shape, device=x.device) for _ in range(2))
        for outs, gs in (((p.log_probs, p.entropy), (g, h)), ((p.log_probs,), (g,)), ((p.entropy,), (h,))):
            got, = torch.autograd.grad(outs, leaf, gs, retain_graph=True)
            zero = torch.zeros_like(g)
            d, da = log_probs64_gradient(x, t, *((g, h) if len(gs) == 2 else (g, zero) if outs[0] is p.log_probs else (zero, h)), ignored)
            z = torch.where(torch.isfinite(lp), lp.abs() / math.log(2), 0.0)
            bound = (U[dtype] + 2 ** -22 * (4 + z) + tol * (2 + math.log(vocab + 1))) * da
            bound = bound + (2 ** -25 if dtype == FP16 else 2 ** -120)   # half of the smallest number; what 2^z flushes
            assert got.shape == x.shape and bool(((got.double() - d).abs() <= bound).all())


def make(rows, vocab, dtype, ignored=False, std=3.0):
    torch.manual_seed(rows * 13 + vocab)
    x = (torch.randn(rows, vocab, device="cuda") * std).to(dtype)
    t = torch.randint(0, vocab, (rows,), device="cuda")
    if ignored:
        t[::3] = -100
    return x, t


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 5, 5), (3, 31, 31), (9, 50, 32), (17, 255, 7), (8, 512, 32), (33, 1000, 3),
                                            (5, 1024, 32), (100, 1025, 20), (7, 4096, 32), (300, 4099, 5), (1, 30522, 5),
                                            (2, 30522, 32), (37, 30522, 10), (617, 30522, 0), (5, 131072, 20), (1, 200001, 32),
                                            (1300, 33278, 20)])
def test_sizes(dtype, rows, vocab, top):
    x, t = make(rows, vocab, dtype, ignored=rows > 4)
    check(x, t, top, gradients=rows * vocab < 20_000_000)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("vocab", [40, 3000, 20000, 70000])
@pytest.mark.parametrize("kind", ["constant", "rising", "falling", "lowest", "few", "plateau", "wide", "zeros of both signs"])
def test_orders_that_are_hard_for_the_alternatives(dtype, vocab, kind):
    x, t = make(6, vocab, dtype)
    if kind == "constant":
        x.fill_(1.5)
    elif kind == "rising":
        x = x.sort(-1).values
    elif kind == "falling":
        x = x.sort(-1, descending=True).values
    elif kind == "lowest":            # the type's lowest value as a mask, of all of a row too
        x[:, ::2] = torch.finfo(dtype).min
        x[1] = torch.finfo(dtype).min
    elif kind == "few":               # fewer than the alternatives that are wanted have a probability
        x[:, 7:] = -math.inf
        x[2] = -math.inf
        t[:] = 3
    elif kind == "plateau":           # many of the largest are equal, and not in the first batch
        x[:, vocab // 2:] = x.amax()
    elif kind == "wide":
        x = (x.float() * 300).to(dtype)
    else:
        x = torch.where(torch.rand(x.shape, device="cuda") < 0.5, 0.0, -0.0).to(dtype)
    for top in (1, 8, 32):
        check(x, t, top, gradients=top == 8)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("vocab", [100, 30522, 100000])
def test_what_is_no_number(dtype, vocab):
    x, t = make(4, vocab, dtype)
    x[0, 17], x[1, 40], x[1, 60], x[2, 50] = math.nan, math.nan, math.nan, math.inf
    p = token_log_probs(x, t, top=3)
    assert torch.isnan(p.log_probs[:3]).all() and torch.isnan(p.entropy[:3]).all() and torch.isnan(p.top_log_probs[:3]).all()
    assert torch.isfinite(p.log_probs[3]) and torch.isfinite(p.entropy[3])
    assert torch.equal(p.top_tokens, likeliest(x, 3))


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_layouts(dtype):
    torch.manual_seed(0)
    x = (torch.randn(5, 9, 3001, device="cuda") * 3).to(dtype)
    t = torch.randint(0, 2990, (5, 9), device="cuda")
    check(x[:, :-1], t[:, 1:], 4)                       # a sequence's next tokens: two strides
    check(x[:, ::2, 1:], t[:, ::2], 4)                  # rows off the boundaries of 16 bytes
    check(x[::2, 3], t[::2, 3], 4)
    check(x.transpose(0, 1), t.t(), 4)
    check(x.transpose(1, 2)[..., :7].contiguous().transpose(1, 2), t[:, :7], 4)   # columns that are not side by side
    check(x[:1, :1].expand(5, 9, 3001), t, 4)
    check(x[0, 0], t[0, 0], 4)
    check(torch.empty(0, 7, device="cuda", dtype=dtype), torch.empty(0, dtype=torch.int64, device="cuda"), 4)
    y = (torch.randn(2, 3, 4, 50, device="cuda")).to(dtype)[:, :2, :3]            # three strides
    check(y, torch.randint(0, 50, (2, 2, 3), device="cuda"), 4)


def loss64(x, t, ignored=-100):
    _, lp, _ = log_probs64(x, t, ignored)
    return -lp.sum(), (t != ignored).sum()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,vocab", [(1, 2), (5, 50), (3000, 40), (9, 1024), (617, 30522), (2, 100000), (4097, 1000)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_cross_entropy(dtype, rows, vocab, reduction):
    x, t = make(rows, vocab, dtype, ignored=rows > 1)
    leaf = x.detach().requires_grad_(True)
    loss = cross_entropy(leaf, t, reduction=reduction)
    total, n = loss64(x, t)
    g = torch.randn(t.shape if reduction == "none" else (), device="cuda")
    if reduction == "none":
        assert torch.equal(loss, -token_log_probs(x, t).log_probs)
        by = -g
    else:
        want = total / n if reduction == "mean" else total
        # each row's bound, and the sums, which are in 64 bits
        assert loss.dtype == FP32 and abs(loss.item() - want.item()) <= (steps(vocab) * 2 ** -24 + 2 ** -21) * (abs(want.item()) + 1)
        by = (-g / n if reduction == "mean" else -g).expand(t.shape)
    got, = torch.autograd.grad(loss, leaf, g)
    d, da = log_probs64_gradient(x, t, by, torch.zeros_like(by))
    z = log_probs64(x, t)[0].abs() / math.log(2)
    bound = (U[dtype] + 2 ** -22 * (8 + z) + steps(vocab) * 2 ** -24) * da + (2 ** -25 if dtype == FP16 else 2 ** -120)
    assert bool(((got.double() - d).abs() <= bound).all())
    assert not got[t == -100].any()


def test_ignored_rows_and_none_at_all():
    x, t = make(6, 2000, BF16)
    x[2], x[3] = math.nan, -math.inf
    t[2] = -100
    leaf = x.detach().requires_grad_(True)
    loss = cross_entropy(leaf, t)
    assert loss == math.inf
    g, = torch.autograd.grad(loss, leaf)
    assert torch.isfinite(g).all() and not g[2].any() and not g[3].any() and g[4].any()
    t.fill_(-100)
    assert math.isnan(cross_entropy(x, t)) and cross_entropy(x, t, reduction="sum") == 0
    assert math.isnan(cross_entropy(x[:0], t[:0])) and cross_entropy(x[:0], t[:0], reduction="sum") == 0
    assert torch.autograd.grad(cross_entropy(leaf[:0], t[:0], reduction="sum"), leaf)[0].shape == leaf.shape


def test_tokens_outside_the_vocabulary():
    x, t = make(4, 500, BF16)
    t[1], t[2] = 500, -1
    leaf = x.detach().requires_grad_(True)
    p = token_log_probs(leaf, t)
    assert torch.isnan(p.log_probs).tolist() == [False, True, True, False] and torch.isfinite(p.entropy).all()
    assert math.isnan(cross_entropy(x, t))
    assert torch.isfinite(token_log_probs(x, t, ignore_index=500).log_probs[1])
    g, = torch.autograd.grad(p.log_probs, leaf, torch.ones_like(p.log_probs))
    assert torch.isnan(g).any(1).tolist() == [False, True, True, False]


def test_more_than_32_bits_of_logits():
    rows, vocab = 70000, 32768
    x = torch.zeros(rows, vocab, dtype=BF16, device="cuda")
    t = torch.full((rows,), 5, device="cuda")
    x[-3:], t[-3:] = (torch.randn(3, vocab, device="cuda") * 3).to(BF16), torch.tensor([0, 1, vocab - 1], device="cuda")
    leaf = x.detach().requires_grad_(True)
    p = token_log_probs(leaf, t, top=2)
    few = x[-3:].clone().requires_grad_(True)
    q = token_log_probs(few, t[-3:], top=2)
    tol = steps(vocab) * 2 ** -24
    assert (p.log_probs[-3:] - q.log_probs).abs().max() <= 2 * tol + 2 ** -20 and torch.equal(p.top_tokens[-3:], q.top_tokens)
    assert (p.log_probs[:-3] + math.log(vocab)).abs().max() <= tol + 2 ** -20
    w = torch.zeros(rows, device="cuda")
    w[-3:] = 1.0
    g, = torch.autograd.grad(p.log_probs, leaf, w)
    want, = torch.autograd.grad(q.log_probs, few, w[-3:])
    assert torch.allclose(g[-3:].float(), want.float(), rtol=2 ** -7, atol=1e-9) and not g[:100].any()


def test_repeatable_streams_and_graphs():
    x, t = make(300, 30522, BF16, ignored=True)
    leaf = x.detach().requires_grad_(True)

    def run(leaf):
        loss = cross_entropy(leaf, t)
        p = token_log_probs(leaf, t, top=10)
        return [loss.detach(), p.log_probs.detach(), p.top_tokens, p.top_log_probs, *torch.autograd.grad((loss, p.entropy.sum()), leaf)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = run(leaf)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(leaf)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, out))
    with torch.no_grad():
        x.copy_(x.flip(0))        # the leaf's own storage
    graph.replay()
    again = run(x.detach().clone().requires_grad_(True))
    assert all(torch.equal(a, b) for a, b in zip(again, out))


def test_refusals_on_the_gpu():
    x, t = make(4, 500, BF16)
    with pytest.raises(ValueError, match="tensors on"):
        token_log_probs(x, t.cpu())
    with pytest.raises(TypeError):
        cross_entropy(x.double(), t)
    leaf = x.detach().requires_grad_(True)
    g, = torch.autograd.grad(cross_entropy(leaf, t), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.float().sum().backward()
    p = token_log_probs(leaf, t, top=3)
    assert not p.top_log_probs.requires_grad and not p.top_tokens.requires_grad
    with torch.no_grad():
        leaf.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        p.log_probs.sum().backward()
