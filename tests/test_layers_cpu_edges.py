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
