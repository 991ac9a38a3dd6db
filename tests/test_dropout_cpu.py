"""Dropout on the CPU: the generator, what its definition says, gradients, refusals."""
import math

import pytest
import torch

from _dropout import attention64, kept, kept_bits, kept_count, kept_probabilities, philox
from _layers import close
from hipress_b200.models import bert_tiny
from hipress_b200.models.bert import BertConfig
from hipress_b200.ops import attention, dropout, layer_norm, self_attention


@pytest.mark.parametrize("rounds,want", [(7, (0x5f6fb709, 0x0d893f64, 0x4f121f81, 0x4f730a48)),
                                         (10, (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8))])
def test_the_generator_is_the_published_one(rounds, want):
    assert tuple(philox((0, 0, 0, 0), (0, 0), rounds)) == want


@pytest.mark.parametrize("seed", [0, 1, -1, 2 ** 63 - 1, -2 ** 63, 123456789012345])
@pytest.mark.parametrize("p,site", [(0.1, 0), (0.5, 7), (0.999, 2 ** 32 - 1), (1e-4, 3)])
def test_elements_are_kept_by_the_definition(seed, p, site):
    n = 3 * 32 + 5
    got = kept((n,), p, seed, site).tolist()
    want = [b for w in range(4) for b in kept_bits(w, seed, site, kept_count(p))][:n]
    assert got == want
    x = torch.randn(n).abs() + 1
    for s in (seed, torch.tensor([seed]), torch.tensor(seed)):
        y = dropout(x, p, seed=s, site=site)
        assert [v != 0 for v in y.tolist()] == want
        assert torch.equal(y, torch.where(torch.tensor(want), x * (65536 / kept_count(p)), 0.0))


def test_probabilities_go_by_rows_of_whole_words():
    b, h, sq, sk = 2, 3, 5, 45
    got = kept_probabilities(b, h, sq, sk, 0.3, 11, 4).reshape(-1, sk)
    for row in (0, 7, b * h * sq - 1):
        assert got[row].tolist() == (kept_bits(2 * row, 11, 4, kept_count(0.3)) + kept_bits(2 * row + 1, 11, 4, kept_count(0.3)))[:sk]


@pytest.mark.parametrize("p", [0.1, 0.5, 0.75, 0.03])
def test_share_and_independence(p):
    n = 1 << 18
    a, b, c = (kept((n,), p, s, t).double() for s, t in ((1, 0), (1, 1), (2, 0)))
    q = kept_count(p) / 65536
    sigma = math.sqrt(q * (1 - q) / n)
    for m in (a, b, c):
        assert abs(m.mean() - q) < 5 * sigma
        for lag in (1, 2, 31, 32, 33, 1024):   # no element says anything of another
            assert abs(((m[lag:] - q) * (m[:-lag] - q)).mean()) < 5 * q * (1 - q) / math.sqrt(n - lag)
    for x, y in ((a, b), (a, c), (b, c)):
        assert abs(((x - q) * (y - q)).mean()) < 5 * q * (1 - q) / math.sqrt(n)


def test_dropped_elements_are_zero_whatever_they_are():
    m = kept((64,), 0.5, 3, 0)
    x = torch.where(m, 1.0, math.nan)
    x[(~m).nonzero()[0]] = math.inf
    y = dropout(x, 0.5, seed=3)
    assert torch.equal(y, torch.where(m, 2.0, 0.0))
    leaf = torch.ones(64, requires_grad=True)
    g, = torch.autograd.grad(dropout(leaf, 0.5, seed=3), leaf, x)
    assert torch.equal(g, y)


def test_gradients_against_differences():
    torch.manual_seed(0)
    x, r = (torch.randn(3, 11, dtype=torch.float64, requires_grad=True) for _ in range(2))
    w, b = (torch.randn(11, dtype=torch.float64, requires_grad=True) for _ in range(2))
    kw = dict(seed=5, site=2)
    assert torch.autograd.gradcheck(lambda x, r: dropout(x, 0.3, residual=r, **kw), (x, r))
    assert torch.autograd.gradcheck(lambda x, w, b, r: layer_norm(x, w, b, residual=r, dropout=0.3, **kw), (x, w, b, r))
    q = torch.randn(2, 5, 4, 3, dtype=torch.float64, requires_grad=True)
    k, v = (torch.randn(2, 7, 2, 3, dtype=torch.float64, requires_grad=True) for _ in range(2))
    mask = torch.arange(7)[None] < torch.tensor([[7], [4]])
    assert torch.autograd.gradcheck(lambda q, k, v: attention(q, k, v, causal=True, key_mask=mask, dropout=0.4, **kw), (q, k, v))


def test_the_layer_norm_drops_what_dropout_drops():
    torch.manual_seed(1)
    x, r, dz = (torch.randn(7, 33) for _ in range(3))
    w = torch.randn(33)
    leaves = [t.clone().requires_grad_(True) for t in (x, r)]
    y, z = layer_norm(leaves[0], w, residual=leaves[1], dropout=0.2, seed=9, site=3)
    assert torch.equal(z, dropout(x, 0.2, seed=9, site=3, residual=r))
    assert torch.equal(y, layer_norm(z, w))
    dx, dr = torch.autograd.grad((y, z), leaves, (torch.zeros_like(y), dz))
    assert torch.equal(dr, dz) and torch.equal(dx, dropout(dz, 0.2, seed=9, site=3))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_attention(dtype):
    torch.manual_seed(2)
    q, do = (torch.randn(2, 9, 4, 8).to(dtype) for _ in range(2))
    k, v = (torch.randn(2, 37, 2, 8).to(dtype) for _ in range(2))
    mask = torch.arange(37)[None] < torch.tensor([[37], [20]])
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    seed = torch.tensor([77])
    o = attention(*leaves, causal=True, key_mask=mask, dropout=0.25, seed=seed, site=1)
    want = attention64(*(t.detach() for t in leaves), do, causal=True, mask=mask, kept=kept_probabilities(2, 4, 9, 37, 0.25, 77, 1),
                       up=65536 / kept_count(0.25))
    close(o, *want["out"], 1, dtype, "out")
    for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)):
        close(g, *want[name], 2, dtype, name)   # delta is made from the rounded result


def test_self_attention_is_attention():
    qkv = torch.randn(2, 6, 3, 2, 4)
    a = self_attention(qkv, dropout=0.5, seed=1, site=9)
    assert torch.equal(a, attention(*qkv.unbind(2), dropout=0.5, seed=1, site=9))
    assert not torch.equal(a, self_attention(qkv, dropout=0.5, seed=1, site=8))


def test_no_dropout_is_none():
    x, r = torch.randn(4, 6), torch.randn(4, 6)
    assert torch.equal(dropout(x, 0.0), x) and torch.equal(dropout(x, 0.0, residual=r), x + r)
    assert torch.equal(dropout(x, 1e-6, seed=None), x)   # less than 2^-17
    assert torch.equal(layer_norm(x, residual=r, dropout=0.0)[0], layer_norm(x, residual=r)[0])
    assert dropout(torch.zeros(0, 5), 0.5, seed=1).shape == (0, 5)
    assert dropout(torch.tensor(3.0), 0.5, seed=1).shape == ()


def test_a_seed_that_moves_between_the_passes_is_refused():
    seed, x = torch.tensor([4]), torch.randn(40, requires_grad=True)
    y = dropout(x, 0.5, seed=seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_second_derivatives_are_refused():
    x = torch.randn(40, requires_grad=True)
    g, = torch.autograd.grad(dropout(x, 0.5, seed=1).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()


def test_refusals():
    x = torch.randn(4, 6)
    for p in (-0.1, 1.0, 1.5, math.nan):
        with pytest.raises(ValueError, match="probability"):
            dropout(x, p, seed=1)
    with pytest.raises(ValueError, match="wants a seed"):
        dropout(x, 0.5)
    for seed in (torch.tensor([1.0]), torch.tensor([1, 2]), torch.tensor([1], dtype=torch.int32)):
        with pytest.raises(TypeError, match="seed"):
            dropout(x, 0.5, seed=seed)
    with pytest.raises(ValueError, match="64 bits"):
        dropout(x, 0.5, seed=2 ** 64)
    for site in (-1, 2 ** 32):
        with pytest.raises(ValueError, match="site"):
            dropout(x, 0.5, seed=1, site=site)
    with pytest.raises(ValueError, match="residual"):
        dropout(x, 0.5, seed=1, residual=x[:2])
    with pytest.raises(ValueError, match="residual"):
        dropout(x, 0.5, seed=1, residual=x.double())
    with pytest.raises(TypeError):
        dropout(x.long(), 0.5, seed=1)
    with pytest.raises(ValueError, match="no residual"):
        layer_norm(x, dropout=0.1, seed=1)
    with pytest.raises(ValueError, match="wants a seed"):
        layer_norm(x, residual=x, dropout=0.1)
    q = torch.randn(2, 4, 3, 8)
    with pytest.raises(ValueError, match="probability"):
        attention(q, q, q, dropout=1.0, seed=1)
    with pytest.raises(ValueError, match="wants a seed"):
        self_attention(torch.randn(2, 4, 3, 2, 8), dropout=0.1)


# ------------------------------------------------------------------------ BERT
def test_bert_on_all_of_the_packages_operators():
    torch.manual_seed(0)
    plain = bert_tiny()
    fused = bert_tiny(fused="all", seed=3)
    fused.load_state_dict(plain.state_dict())
    ids = torch.randint(0, 1000, (3, 40))
    labels = torch.where(torch.rand(3, 40) < 0.3, ids, -100)
    a, b = fused(ids, labels).item(), fused(ids, labels).item()
    assert a != b                                    # a pass of its own, a mask of its own
    fused.drop_seed.fill_(3)
    assert fused(ids, labels).item() == a            # the same seed, the same masks
    plain.eval(), fused.eval()
    assert abs(fused(ids, labels) - plain(ids, labels)) < 1e-5 * abs(plain(ids, labels))
    p = fused.score(ids, labels, top=3)
    lp = torch.log_softmax(fused(ids), -1)[labels != -100]
    assert torch.allclose(p.log_probs, lp.gather(1, labels[labels != -100][:, None])[:, 0], atol=1e-5)
    assert torch.allclose(p.top_log_probs, lp.topk(3).values, atol=1e-5)
    assert torch.allclose(-p.log_probs.mean(), fused(ids, labels), atol=1e-5)
    with pytest.raises(ValueError, match="fused"):
        BertConfig(fused="some")
    assert BertConfig(fused="all").attn_dropout == 0.1


def test_two_passes_before_the_first_backward_pass():
    m = bert_tiny(fused="all")
    ids = torch.randint(0, 1000, (2, 8))
    (m(ids, ids) + m(ids, ids)).backward()   # each has a seed of its own, which stays
    assert all(p.grad is None or torch.isfinite(p.grad).all() for p in m.parameters())
