"""The layer operators' kernels value by value, where a norm over the whole result shows nothing:
tails of the activations, infinities that a rounding made, gradients far below one."""
import math

import pytest
import torch

from _layers import U, act64

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
