"""The layer operators on CPU tensors at the ends of their range."""
import pytest
import torch

from hipress_b200.ops import linear


@pytest.mark.parametrize("lead", [(4,), (2, 3), (0, 3), (2, 0, 1), ()])
@pytest.mark.parametrize("k,n", [(0, 8), (16, 0), (0, 0)])
def test_linear_empty_sizes_of_any_shape(lead, k, n):
    x, w = torch.randn(*lead, k, requires_grad=True), torch.randn(n, k, requires_grad=True)
    b, r = torch.randn(n, requires_grad=True), torch.randn(*lead, n, requires_grad=True)
    y = linear(x, w, b, activation="relu", residual=r)
    assert y.shape == (*lead, n)
    if k == 0:
        assert torch.equal(y, b.clamp(min=0) + r)
    dx, dw, db, dr = torch.autograd.grad(y, (x, w, b, r), torch.ones_like(y))
    assert dx.shape == x.shape and not dx.any() and dw.shape == w.shape and not dw.any()
    assert db.shape == b.shape and torch.equal(dr, torch.ones_like(dr))


@pytest.mark.parametrize("kind", ["relu", "gelu", "gelu_tanh"])
def test_slope_at_an_infinity_that_only_the_rounding_made(kind):
    """In front of the activation -90000 and 90000 become infinities of fp16."""
    x = torch.tensor([[300.0, 0.0], [-300.0, 0.0], [1.0, 1.0]], dtype=torch.float16, requires_grad=True)
    w = torch.tensor([[300.0, 2.0]], dtype=torch.float16, requires_grad=True)
    b = torch.zeros(1, requires_grad=True)
    y = linear(x, w, b, activation=kind)
    assert y[1].item() == 0
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.tensor([[0.5], [1.0], [0.25]], dtype=torch.float16))
    assert torch.equal(dx, torch.tensor([[150.0, 1.0], [0.0, 0.0], [75.0, 0.5]], dtype=torch.float16))
    assert torch.equal(dw, torch.tensor([[150.25, 0.25]], dtype=torch.float16)) and db.item() == 0.75


@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh"])
def test_slope_of_very_large_values(kind):
    x = torch.tensor([[3e38], [1e20], [-1e20], [-3e38]], requires_grad=True)
    y = linear(x, torch.ones(1, 1), activation=kind)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert dx.flatten().tolist() == [1.0, 1.0, 0.0, 0.0] and (y[2:] == 0).all()
