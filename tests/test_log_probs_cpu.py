"""Log probabilities of tokens and the cross entropy on the CPU: formulas, edges, gradients, refusals."""
import math

import pytest
import torch
import torch.nn.functional as F

from _dropout import likeliest, log_probs64, log_probs64_gradient
from hipress_b200.ops import TokenLogProbs, cross_entropy, token_log_probs


def case(rows=5, vocab=37, dtype=torch.float32):
    torch.manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab) * 3).to(dtype)
    t = torch.randint(0, vocab, (rows,))
    t[1] = -100
    return x, t


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
def test_formulas(dtype):
    x, t = case(dtype=dtype)
    got = token_log_probs(x, t, top=4)
    lp, want, entropy = log_probs64(x, t)
    assert isinstance(got, TokenLogProbs) and got.log_probs.dtype == (torch.float64 if dtype == torch.float64 else torch.float32)
    assert torch.allclose(got.log_probs.double(), want, atol=1e-5) and torch.allclose(got.entropy.double(), entropy, atol=1e-5)
    best = likeliest(x, 4)
    assert torch.equal(got.top_tokens, best) and torch.allclose(got.top_log_probs.double(), lp.gather(1, best), atol=1e-5)
    assert token_log_probs(x, t)[2:] == (None, None) and token_log_probs(x, t, entropy=False).entropy is None
    for reduction in ("mean", "sum", "none"):
        ours = cross_entropy(x, t, reduction=reduction)
        assert torch.allclose(ours.double(), F.cross_entropy(x.double(), t, reduction=reduction), atol=1e-5)


def test_gradients_against_differences_and_the_formula():
    x, t = case(dtype=torch.float64)
    x.requires_grad_(True)
    assert torch.autograd.gradcheck(lambda x: token_log_probs(x, t)[:2], (x,))
    for reduction in ("mean", "sum", "none"):
        assert torch.autograd.gradcheck(lambda x: cross_entropy(x, t, reduction=reduction), (x,))
    g, h = torch.randn(5, dtype=torch.float64), torch.randn(5, dtype=torch.float64)
    got, = torch.autograd.grad(token_log_probs(x, t)[:2], x, (g, h))
    assert torch.allclose(got, log_probs64_gradient(x.detach(), t, g, h)[0])
    tops = token_log_probs(x, t, top=3)
    assert not tops.top_log_probs.requires_grad and not tops.top_tokens.requires_grad


def test_rows_with_nothing_and_ignored_rows():
    x, t = case()
    x[0] = -math.inf
    x[2, 5:] = -math.inf
    t[2] = 3
    x[1] = math.nan                # ignored: no gradient, whatever it holds
    leaf = x.clone().requires_grad_(True)
    p = token_log_probs(leaf, t, top=3)
    assert p.log_probs[0] == -math.inf and p.entropy[0] == 0 and p.log_probs[1] == 0
    assert p.top_tokens[0].tolist() == [0, 1, 2] and (p.top_log_probs[0] == -math.inf).all()
    assert torch.isfinite(p.entropy[2]) and torch.isfinite(p.log_probs[2])
    loss = cross_entropy(leaf, t)
    assert loss == math.inf
    g, = torch.autograd.grad(loss, leaf)
    assert torch.isfinite(g).all() and not g[0].any() and not g[1].any() and g[2].any()
    assert math.isnan(cross_entropy(x, torch.full_like(t, -100)))
    assert cross_entropy(x, torch.full_like(t, -100), reduction="sum") == 0


def test_logits_at_the_types_lowest_value():
    low = torch.finfo(torch.bfloat16).min
    x = torch.full((2, 8), low, dtype=torch.bfloat16)
    x[1, 2:4] = 1.0
    p = token_log_probs(x, torch.tensor([3, 3]))
    assert torch.allclose(p.log_probs, torch.tensor([-math.log(8), -math.log(2)]))
    assert torch.allclose(p.entropy, torch.tensor([math.log(8), math.log(2)]))


def test_equal_values_count_from_the_lowest_place():
    x = torch.tensor([[1.0, 3.0, 3.0, 0.0, -0.0, 3.0], [0.0, -0.0, 0.0, -0.0, 0.0, 0.0]])
    p = token_log_probs(x, torch.tensor([0, 0]), top=5)
    assert p.top_tokens.tolist() == [[1, 2, 5, 0, 3], [0, 1, 2, 3, 4]]


def test_shapes():
    x = torch.randn(2, 3, 7)
    t = torch.randint(0, 7, (2, 3))
    assert [a.shape for a in token_log_probs(x, t, top=2)] == [(2, 3), (2, 3), (2, 3, 2), (2, 3, 2)]
    assert token_log_probs(x[0, 0], t[0, 0], top=1).top_tokens.shape == (1,)
    assert cross_entropy(x[:, :0], t[:, :0], reduction="none").shape == (2, 0)
    assert math.isnan(cross_entropy(x[:, :0], t[:, :0]))


def test_refusals():
    x, t = case()
    with pytest.raises(ValueError, match="int64"):
        token_log_probs(x, t.int())
    with pytest.raises(ValueError, match="int64"):
        token_log_probs(x, t[:2])
    with pytest.raises(TypeError):
        token_log_probs(x.long(), t)
    for top in (-1, 33, 38):
        with pytest.raises(ValueError, match="likeliest"):
            token_log_probs(x, t, top=top)
    with pytest.raises(ValueError, match="vocabulary"):
        token_log_probs(x[:, :0], t)
    with pytest.raises(ValueError, match="vocabulary"):
        token_log_probs(torch.tensor(1.0), torch.tensor(0))
    with pytest.raises(ValueError, match="reduction"):
        cross_entropy(x, t, reduction="median")
    t[0] = 37
    with pytest.raises(IndexError, match="37"):
        cross_entropy(x, t)
    leaf = x.requires_grad_(True)
    t[0] = 0
    g, = torch.autograd.grad(cross_entropy(leaf, t), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()
