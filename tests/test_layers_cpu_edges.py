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


def operators(device, dtype):
    """Each operator and the leaves of one call."""
    from hipress_b200.ops import attention, layer_norm, self_attention
    torch.manual_seed(7)
    g = lambda *s: torch.randn(*s, device=device).to(dtype).requires_grad_(True)  # noqa: E731
    x, r, nw, lw, q, k, qkv = g(6, 16), g(6, 16), g(16), g(8, 16), g(1, 5, 2, 8), g(1, 7, 2, 8), g(1, 5, 3, 2, 8)
    return {"layer_norm": (lambda: layer_norm(x, nw), (x, nw)),
            "layer_norm residual": (lambda: sum(layer_norm(x, nw, residual=r)), (x, nw, r)),
            "linear": (lambda: linear(x, lw), (x, lw)), "linear gelu": (lambda: linear(x, lw, activation="gelu"), (x, lw)),
            "attention": (lambda: attention(q, k, k), (q, k)), "self_attention": (lambda: self_attention(qkv), (qkv,))}


def check_second_derivatives(device, dtype, name):
    """They are refused, also where the gradient that comes in is a constant; the first ones are not."""
    call, leaves = operators(device, dtype)[name]
    want = torch.autograd.grad(call().sum(), leaves)
    got = torch.autograd.grad(call().sum(), leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    penalty = sum(t.float().square().sum() for t in got)
    with pytest.raises(RuntimeError, match="differentiate"):
        torch.autograd.grad(call().float().square().sum() + penalty, leaves)
    got = torch.autograd.grad(call().float().square().sum(), leaves, create_graph=True)   # a gradient that has one itself
    with pytest.raises(RuntimeError, match="differentiate"):
        torch.autograd.grad(got[0].float().square().sum(), leaves[0])


OPERATORS = ["layer_norm", "layer_norm residual", "linear", "linear gelu", "attention", "self_attention"]


@pytest.mark.parametrize("name", OPERATORS)
def test_second_derivatives_are_refused(name):
    check_second_derivatives("cpu", torch.float32, name)
