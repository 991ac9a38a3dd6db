"""The layer operators' kernels row by row against 64 bits, within bounds that a lost row, a lost
tile or a wrong factor breaks (tests/test_layers_bounds.py shows that)."""
import pytest
import torch

from _layers_rows import attention_rows, linear_rows, off
from test_gpu_layers import MANY, SHAPES, SIZES, rand

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def mask_of(kind, b, sk):
    if kind is None:
        return None
    if kind == "holes":
        return torch.rand(b, sk, device="cuda") < 0.6
    mask = torch.arange(sk, device="cuda")[None] < torch.randint(0, sk + 1, (b, 1), device="cuda")
    mask[0] = False            # a sequence of which nothing is left
    return mask


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("masked", [None, "lengths", "holes"])
@pytest.mark.parametrize("shape", SHAPES + MANY + [(1, 1500, 1500, 2, 1, 64), (1, 1031, 2055, 4, 2, 128), (2, 640, 640, 3, 3, 32)])
def test_attention_by_rows(dtype, causal, masked, shape):
    from hipress_b200.ops import attention
    b, sq, sk, h, hk, d = shape
    torch.manual_seed(sq + 3 * sk + d)
    q, do = rand(b, sq, h, d, dtype=dtype), rand(b, sq, h, d, dtype=dtype)
    k, v = rand(b, sk, hk, d, dtype=dtype), rand(b, sk, hk, d, dtype=dtype)
    mask = mask_of(masked, b, sk)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = attention(*leaves, causal=causal, key_mask=mask)
    got = (out, *torch.autograd.grad(out, leaves, do))
    for (name, (exact, bound)), g in zip(attention_rows(q, k, v, do, causal=causal, mask=mask).items(), got):
        assert off(g, exact, bound) <= 1, name


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("scale", [0.0, -0.3, 0.9])
@pytest.mark.parametrize("shape", [(2, 100, 120, 2, 2, 64), (1, 300, 500, 4, 2, 64), (1, 300, 260, 2, 2, 128)])
def test_attention_by_rows_of_other_scales(dtype, scale, shape):
    from hipress_b200.ops import attention
    b, sq, sk, h, hk, d = shape
    torch.manual_seed(sq)
    q, do = rand(b, sq, h, d, dtype=dtype), rand(b, sq, h, d, dtype=dtype)
    k, v = rand(b, sk, hk, d, dtype=dtype), rand(b, sk, hk, d, dtype=dtype)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = attention(*leaves, scale=scale)
    got = (out, *torch.autograd.grad(out, leaves, do))
    for (name, (exact, bound)), g in zip(attention_rows(q, k, v, do, scale=scale).items(), got):
        assert off(g, exact, bound) <= 1, name


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("sq,sk", [(1, 65), (65, 129), (129, 193), (200, 513), (513, 1025), (130, 127)])
def test_attention_ends_count(dtype, dim, sq, sk):
    """The last key takes half of every row, the last query half of every key's gradient: a tail that
    is lost, however short, shows in all rows."""
    from hipress_b200.ops import attention
    torch.manual_seed(sk + dim)
    q, k, v, do = (rand(1, s, 2, dim, dtype=FP32, std=0.3) for s in (sq, sk, sk, sq))
    lean = torch.randn(dim, device="cuda").sign()
    q += lean
    k[:, -1] += lean * torch.log(torch.tensor(float(sk))) / dim ** 0.5
    v[:, -1] += 1
    do[:, -1] *= sq ** 0.5
    q, k, v, do = (t.to(dtype) for t in (q, k, v, do))
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = attention(*leaves)
    got = (out, *torch.autograd.grad(out, leaves, do))
    rows = attention_rows(q, k, v, do)
    for (name, (exact, bound)), g in zip(rows.items(), got):
        assert off(g, exact, bound) <= 1, name
    without = {**attention_rows(q, k[:, :-1], v[:, :-1], do), **{n: r for n, r in attention_rows(q[:, :-1], k, v, do[:, :-1]).items()
                                                                   if n in ("dk", "dv")}} if sq > 1 else {}
    for name, (exact, bound) in rows.items():
        if name in without and without[name][0].shape == exact.shape:
            assert (without[name][0] - exact).norm(dim=-1).gt(bound).float().mean() > 0.5, name


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("kind", [None, "relu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear_by_rows(dtype, kind, m, k, n):
    from hipress_b200.ops import linear
    torch.manual_seed(m + 3 * k + n)
    for wtype, residual in ((dtype, False), (FP32, True)):
        x, w, b = rand(m, k, dtype=dtype), rand(n, k, dtype=wtype, std=k ** -0.5), rand(n, dtype=wtype)
        r, dy = rand(m, n, dtype=dtype) if residual else None, rand(m, n, dtype=dtype)
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = linear(*leaves, activation=kind, residual=r)
        got = dict(zip(("y", "dx", "dw", "db"), (y, *torch.autograd.grad(y, leaves, dy))))
        for name, (exact, bound) in linear_rows(x, w, b, r, dy, kind).items():
            assert off(got[name], exact, bound) <= 1, name
