"""The layer operators on CPU tensors: formulas, gradients against differences, refusals."""
import math

import pytest
import torch
import torch.nn.functional as F

from hipress_b200.ops import attention, layer_norm, linear, self_attention

from _layers import attention64, close, linear64, norm64

F64 = torch.float64


def rand(*shape, dtype=F64):
    return torch.randn(*shape, dtype=F64).to(dtype).requires_grad_(True)


def test_layer_norm_gradient_against_differences():
    torch.manual_seed(0)
    x, r, w, b = rand(3, 5, 7), rand(3, 5, 7), rand(7), rand(7)
    assert torch.autograd.gradcheck(layer_norm, (x, w, b))
    assert torch.autograd.gradcheck(lambda x, w, b, r: layer_norm(x, w, b, residual=r), (x, w, b, r))
    assert torch.autograd.gradcheck(lambda x, r: layer_norm(x, residual=r)[1], (x, r))


@pytest.mark.parametrize("kind", [None, "relu", "gelu", "gelu_tanh"])
def test_linear_gradient_against_differences(kind):
    torch.manual_seed(1)
    args = rand(4, 6), rand(5, 6), rand(5), rand(4, 5)
    assert torch.autograd.gradcheck(lambda x, w, b, r: linear(x, w, b, activation=kind, residual=r), args)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("sq,sk", [(5, 5), (3, 6), (6, 3)])
def test_attention_gradient_against_differences(causal, sq, sk):
    torch.manual_seed(2)
    q, k, v = rand(2, sq, 4, 3), rand(2, sk, 2, 3), rand(2, sk, 2, 3)
    mask = torch.rand(2, sk) < 0.7
    mask[0, :2] = False
    assert torch.autograd.gradcheck(lambda q, k, v: attention(q, k, v, causal=causal, key_mask=mask), (q, k, v))


def test_self_attention_gradient_against_differences():
    torch.manual_seed(3)
    assert torch.autograd.gradcheck(lambda t: self_attention(t, causal=True), (rand(2, 4, 3, 2, 5),))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_formulas(dtype):
    """What a model gets is what torch's own layers compute, and what the oracle computes."""
    torch.manual_seed(4)
    x, w, b, dy = (rand(*s, dtype=dtype) for s in ((9, 16), (16,), (16,), (9, 16)))
    y = layer_norm(x, w, b)
    want = norm64(x.detach(), w.detach(), b.detach(), dy.detach(), None, 1e-5)
    close(y, *want["y"], 1, dtype, "y")
    for name, g in zip(("dx", "dw", "db"), torch.autograd.grad(y, (x, w, b), dy)):
        close(g, *want[name], 1, dtype, name)
    assert torch.allclose(y, F.layer_norm(x, (16,), w, b), rtol=2 ** -7, atol=2 ** -7)
    x, w, b, r, dy = (rand(*s, dtype=dtype) for s in ((9, 16), (12, 16), (12,), (9, 12), (9, 12)))
    y = linear(x, w, b, activation="gelu", residual=r)
    want = linear64(*(t.detach() for t in (x, w, b, r, dy)), "gelu")
    close(y, *want["y"], 1, dtype, "y")
    for name, g in zip(("dx", "dw", "db"), torch.autograd.grad(y, (x, w, b), dy)):
        close(g, *want[name], 3, dtype, name)
    q, k, v, do = (rand(2, 7, 3, 8, dtype=dtype) for _ in range(4))
    o, lse = attention(q, k, v, causal=True, return_lse=True)
    want = attention64(*(t.detach() for t in (q, k, v, do)), causal=True, mask=None)
    close(o, *want["out"], 1, dtype, "out")
    assert not lse.requires_grad and torch.allclose(lse.double(), want["lse"][0], atol=1e-5)
    for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)):
        close(g, *want[name], 2, dtype, name)
    t = lambda x: x.transpose(1, 2)  # noqa: E731
    sdpa = t(F.scaled_dot_product_attention(t(q), t(k), t(v), is_causal=True))
    assert torch.allclose(o, sdpa, rtol=2 ** -6, atol=2 ** -6)


def test_rows_that_see_nothing_and_what_masked_keys_hold():
    torch.manual_seed(5)
    q, k, v = (torch.randn(1, s, 2, 4) for s in (6, 3, 3))
    mask = torch.tensor([[False, True, True]])
    k[:, 0], v[:, 0] = math.nan, math.inf
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    o, lse = attention(*leaves, causal=True, key_mask=mask, return_lse=True)
    assert not o[:, :4].any() and (lse[:, :, :4] == -math.inf).all() and torch.isfinite(o).all()
    for g in torch.autograd.grad(o, leaves, torch.ones_like(o)):
        assert torch.isfinite(g).all()


def test_refusals():
    x, w = torch.randn(4, 6), torch.randn(5, 6)
    with pytest.raises(ValueError, match="columns"):
        layer_norm(x, torch.ones(5))
    with pytest.raises(ValueError, match="residual"):
        layer_norm(x, residual=x[:2])
    with pytest.raises(TypeError):
        layer_norm(x.long())
    with pytest.raises(TypeError):
        layer_norm(x, torch.ones(6, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="no columns"):
        layer_norm(torch.zeros(3, 0))
    with pytest.raises(ValueError, match="activation"):
        linear(x, w, activation="swish")
    with pytest.raises(ValueError, match="shape"):
        linear(x, w.t())
    with pytest.raises(ValueError, match="bias"):
        linear(x, w, torch.ones(6))
    with pytest.raises(ValueError, match="residual"):
        linear(x, w, residual=x)
    q = torch.randn(2, 4, 3, 8)
    with pytest.raises(ValueError, match="heads"):
        attention(q, q[:, :, :2], q[:, :, :2])
    with pytest.raises(ValueError, match="alike"):
        attention(q, q, q[:, :3])
    with pytest.raises(TypeError):
        attention(q, q, q.double())
    with pytest.raises(ValueError, match="key_mask"):
        attention(q, q, q, key_mask=torch.ones(2, 4))
    with pytest.raises(ValueError, match="key_mask"):
        attention(q, q, q, key_mask=torch.ones(2, 5, dtype=torch.bool))
    with pytest.raises(ValueError, match="scale"):
        attention(q, q, q, scale=math.inf)
    with pytest.raises(ValueError, match="batch, length, 3"):
        self_attention(q)
