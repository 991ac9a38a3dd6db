"""The layer operators' kernels value by value, where a norm over the whole result shows nothing:
tails of the activations, infinities that a rounding made, gradients far below one."""
import math

import pytest
import torch

from _layers import U, act64, attention64, norm64

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def rand(*shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(*shape, device="cuda") * std + mean).to(dtype)


def test_linear_empty_sizes_of_any_shape():
    from hipress_b200.ops import linear
    for lead in ((4,), (2, 3), (0, 3), (2, 0, 1), ()):
        for k, n in ((0, 8), (16, 0), (0, 0)):
            x, w = rand(*lead, k, dtype=BF16).requires_grad_(True), rand(n, k, dtype=BF16).requires_grad_(True)
            b, r = rand(n, dtype=BF16).requires_grad_(True), rand(*lead, n, dtype=BF16).requires_grad_(True)
            y = linear(x, w, b, activation="relu", residual=r)
            assert y.shape == (*lead, n)
            if k == 0:
                assert torch.equal(y, (b.float().clamp(min=0) + r.float()).to(BF16))
            dx, dw, db, dr = torch.autograd.grad(y, (x, w, b, r), torch.ones_like(y))
            assert dx.shape == x.shape and not dx.any() and dw.shape == w.shape and not dw.any()
            assert db.shape == b.shape and torch.equal(dr, torch.ones_like(dr))


def one_by_one(values, kind):
    """activation(x) and its derivative of each value, through a product over one k."""
    from hipress_b200.ops import linear
    x = values[:, None].detach().requires_grad_(True)
    y = linear(x, torch.ones(1, 1, device="cuda", dtype=values.dtype), activation=kind)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    return y[:, 0].detach(), dx[:, 0]


@pytest.mark.parametrize("kind", ["relu", "gelu", "gelu_tanh"])
def test_slope_at_an_infinity_that_only_the_rounding_made(kind):
    """In front of the activation -90000 and 90000 become infinities of fp16."""
    from hipress_b200.ops import linear
    x = torch.tensor([[300.0, 0.0], [-300.0, 0.0], [1.0, 1.0]], device="cuda", dtype=FP16).requires_grad_(True)
    w = torch.tensor([[300.0, 2.0]], device="cuda", dtype=FP16).requires_grad_(True)
    b = torch.zeros(1, device="cuda", dtype=FP32, requires_grad=True)
    y = linear(x, w, b, activation=kind)
    assert y[1].item() == 0
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.tensor([[0.5], [1.0], [0.25]], device="cuda", dtype=FP16))
    assert torch.equal(dx, torch.tensor([[150.0, 1.0], [0.0, 0.0], [75.0, 0.5]], device="cuda", dtype=FP16))
    assert torch.equal(dw, torch.tensor([[150.25, 0.25]], device="cuda", dtype=FP16)) and db.item() == 0.75


@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh"])
def test_slope_of_very_large_values(kind):
    y, dx = one_by_one(torch.tensor([3e38, 1e20, -1e20, -3e38], device="cuda", dtype=BF16), kind)
    assert dx.tolist() == [1.0, 1.0, 0.0, 0.0] and (y[2:] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_gelu_is_rounded_once(dtype):
    """All values from -13 to 13.  Besides the result's rounding: the formula's relative error, and
    that of exp(-p p / 2), whose exponent of up to 122 is rounded to 32 bits (122 2^-24 < 2^-17)."""
    bits = torch.arange(-32768, 32768, device="cuda", dtype=torch.int32).to(torch.int16)
    p = bits.view(dtype)
    p = p[torch.isfinite(p) & (p.abs() <= 13)].contiguous()
    y, dx = one_by_one(p, "gelu")
    want, slope = act64(p.double(), "gelu")
    least = {BF16: 2.0 ** -126, FP16: 2.0 ** -24}[dtype]   # half of the smallest number, or what counts as none
    off = ((y.double() - want).abs() - least).clamp(min=0) / want.abs().clamp(min=least)
    assert off.max() <= U[dtype] + 2.0 ** -14, (off.max().item(), p[off.argmax()].item())
    # the derivative is a sum of two terms, which cancel near -0.75
    tail = 0.5 * torch.special.erfc(-p.double() / math.sqrt(2))
    scale = tail + p.double().abs() * torch.exp(-p.double() ** 2 / 2) / math.sqrt(2 * math.pi)
    off = ((dx.double() - slope).abs() - U[dtype] * slope.abs() - least).clamp(min=0) / scale.clamp(min=least)
    assert off.max() <= 2.0 ** -14, (off.max().item(), p[off.argmax()].item())


def heads64(q, k, v, do, scale):
    """dq, dk, dv of one head each in 64 bits, by rows of queries."""
    q, k, v, do = (t.double().transpose(1, 2) for t in (q, k, v, do))
    p = torch.softmax(q @ k.transpose(2, 3) * scale, -1)
    dp = do @ v.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    return tuple(t.transpose(1, 2) for t in (ds @ k, ds.transpose(2, 3) @ q, p.transpose(2, 3) @ do))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("sq,sk", [(100, 128), (300, 8000), (3000, 20000), (257, 20000)])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -10, 2.0 ** 9])
def test_attention_small_gradients_over_long_rows(dim, sq, sk, size):
    """Probabilities of 1 / 20000 times small gradients are below fp16's smallest number long before
    the sums over them are; nothing may become zero, or infinite, on the way."""
    from hipress_b200.ops import attention
    torch.manual_seed(dim + sk)
    lean = torch.randn(1, 1, 1, dim, device="cuda")
    q = rand(1, sq, 1, dim, dtype=FP16, std=0.3)
    # keys and values lean one way, so that sums over them do not cancel
    side = torch.sign(torch.randn(1, sk, 1, 1, device="cuda"))
    k = (rand(1, sk, 1, dim, dtype=FP32, std=0.3) + 2 * side * lean).to(FP16)
    v = (rand(1, sk, 1, dim, dtype=FP32, std=0.3) + side).to(FP16)
    do = ((rand(1, sq, 1, dim, dtype=FP32) * 0.1 + 1) * size * 2.0 ** -6).to(FP16)
    q = (q.float() - (q.float() * lean).sum(-1, keepdim=True) * lean / (lean * lean).sum()).to(FP16)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(attention(*leaves, scale=dim ** -0.5), leaves, do)
    for name, g, want in zip(("dq", "dk", "dv"), got, heads64(q, k, v, do, dim ** -0.5)):
        # results down to fp16's smallest numbers: each within a unit of those besides its share of the whole
        bound = 4 * U[FP16] * want.norm() + math.sqrt(g.numel()) * 2.0 ** -25
        assert (g.double() - want).norm() <= bound, (name, ((g.double() - want).norm() / want.norm()).item())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("sq,sk,causal", [(90, 120, False), (600, 5000, True), (1300, 700, False)])
def test_attention_rows_of_very_unlike_gradients(dim, sq, sk, causal):
    """Each query's dq by itself, where rows of d_o lie up to 2^16 apart, and shared key heads."""
    from hipress_b200.ops import attention
    torch.manual_seed(sq)
    q, k, v = rand(1, sq, 4, dim, dtype=FP16, std=0.5), rand(1, sk, 2, dim, dtype=FP16), rand(1, sk, 2, dim, dtype=FP16)
    power = torch.randint(-12, 5, (1, sq, 1, 1), device="cuda").float()
    do = (rand(1, sq, 4, dim, dtype=FP32) * 2 ** power).to(FP16)
    do[0, sq // 2] = 0
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(attention(*leaves, causal=causal), leaves, do)
    want = attention64(q, k, v, do, causal=causal, mask=None)
    # a row's share of its own sums of absolute values: dS, delta from the rounded result, dq itself.  The
    # short kernel has one factor for all rows: 2^-25 of the largest of them, for each key
    exact, scale = want["dq"]
    worst = ((dq.double() - exact).norm(dim=-1) - dim ** 0.5 * 2.0 ** -25).clamp(min=0)
    allowed = (3 * U[FP16] + 2.0 ** -13) * scale.norm(dim=-1)
    if sq <= 128 and dim <= 64:
        largest = 2 * do.double().norm(dim=-1).amax()
        allowed = allowed + 2.0 ** -25 * largest * k.double().norm(dim=-1).amax() * sk ** 0.5 * dim ** -0.5
    assert (worst <= allowed).all(), (worst / allowed.clamp(min=1e-30)).max().item()
    assert not dq[0, sq // 2].any()
    for name, got in (("dk", dk), ("dv", dv)):
        exact, scale = want[name]
        assert (got.double() - exact).norm() <= (3 * U[FP16] + 2.0 ** -13) * scale.norm(), name


def test_attention_gradients_at_the_end_of_the_range():
    """Gradients scaled up for fp16's sake, and values near 200: neither result nor dS may become infinite."""
    from hipress_b200.ops import attention
    torch.manual_seed(3)
    for sq, sk, dim in ((100, 100, 64), (500, 700, 64), (300, 400, 128)):
        q, k = rand(1, sq, 2, dim, dtype=FP16, std=0.2), rand(1, sk, 2, dim, dtype=FP16, std=0.2)
        v = rand(1, sk, 2, dim, dtype=FP16, std=200)
        do = rand(1, sq, 2, dim, dtype=FP16, std=0.25)
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        got = torch.autograd.grad(attention(*leaves), leaves, do)
        want = attention64(q, k, v, do, causal=False, mask=None)
        for name, g in zip(("dq", "dk", "dv"), got):
            assert torch.isfinite(g).all()
            assert (g.double() - want[name][0]).norm() <= (3 * U[FP16] + 2.0 ** -13) * want[name][1].norm(), name


# lengths at which the ring and the weights together come within a few bytes of the shared memory that a CTA may have
FULL = [(BF16, c) for c in (1954, 2490, 2497, 2613, 2617, 3944, 5009, 5528, 6482, 7896, 10034, 11041, 12280, 13816, 15777)] + \
    [(FP32, c) for c in (460, 628, 677, 1228, 1245, 1305, 3948, 4252, 6140, 6908, 7889)]


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype,cols", FULL)
def test_layer_norm_lengths_that_fill_shared_memory(dtype, cols, residual):
    from hipress_b200.ops import layer_norm
    torch.manual_seed(cols)
    rows = 37
    x, dy, dz = (rand(rows, cols, dtype=dtype) for _ in range(3))
    r = rand(rows, cols, dtype=dtype) if residual else None
    w, b = rand(cols, dtype=FP32, mean=1), rand(cols, dtype=FP32)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    out = layer_norm(*leaves, residual=r)
    z = (x.float() + r.float()).to(dtype) if residual else x
    dx, dw, db = torch.autograd.grad(out, leaves, (dy, dz) if residual else dy)
    want = norm64(z, w, b, dy, dz if residual else None, 1e-5)
    steps = 64 + cols // 32
    for name, got, kind in (("y", out[0] if residual else out, dtype), ("dx", dx, dtype), ("dw", dw, FP32), ("db", db, FP32)):
        exact, scale = want[name]
        assert ((got.double() - exact).abs() <= U[kind] * exact.abs() + steps * 2.0 ** -23 * scale.abs().amax(-1, keepdim=True)).all(), name


def test_attention_gradients_of_scores_that_32_bits_cannot_hold():
    """Scores of 10^7: the probabilities are those of rounded scores, and every gradient a number."""
    from hipress_b200.ops import attention
    torch.manual_seed(8)
    for sq, sk, dim in ((100, 128, 64), (300, 500, 64), (300, 260, 128)):
        q, k = rand(1, sq, 1, dim, dtype=FP16, std=3000), rand(1, sk, 1, dim, dtype=FP16, std=3000)
        v, do = rand(1, sk, 1, dim, dtype=FP16), rand(1, sq, 1, dim, dtype=FP16, std=2.0 ** -10)
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = attention(*leaves)
        for t in (out, *torch.autograd.grad(out, leaves, do)):
            assert torch.isfinite(t).all()
