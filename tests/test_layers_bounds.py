"""What the bounds of tests/_layers_rows.py let through: results rounded as the kernels round them, and
none with a row, a tile, a term or a factor wrong."""
import pytest
import torch

from _layers import act64, attention64, linear64
from _layers_rows import attention_rows, linear_rows, off
from test_gpu_layers import SHAPES, SIZES

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
# sequences and heads beyond the first few show nothing more
SMALL = [(min(b, 2), sq, sk, h if h == hk else 2 * (h // hk), 2 if h != hk else hk, d) for b, sq, sk, h, hk, d in SHAPES]


def rand(*shape, dtype, std=1.0):
    return (torch.randn(*shape) * std).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SMALL)
def test_attention_bounds(dtype, causal, shape):
    b, sq, sk, h, hk, d = shape
    torch.manual_seed(sq + sk)
    q, do = rand(b, sq, h, d, dtype=dtype), rand(b, sq, h, d, dtype=dtype)
    k, v = rand(b, sk, hk, d, dtype=dtype), rand(b, sk, hk, d, dtype=dtype)
    rows = attention_rows(q, k, v, do, causal=causal)
    # the last whole tile of keys, or the last queries, left out (one key of many alone is within the rounding:
    # where it counts for itself is a test of its own)
    keys = (torch.arange(sk) < (sk // 64 - 1) * 64) | (torch.arange(sk) >= sk // 64 * 64)
    less_keys = attention64(q, k, v, do, causal=causal, mask=keys.expand(b, sk)) if sk > 64 else None
    cut = (sq - 1) // 64 * 64
    less_queries = attention64(q, k, v, torch.where((torch.arange(sq) < cut)[:, None, None], do, 0.0), causal=causal, mask=None) \
        if cut else None
    for name, (exact, bound) in rows.items():
        assert off(exact.to(dtype), exact, bound) <= 1, name
        if not (exact.norm(dim=-1) > 8 * bound).any():   # of one key there are no gradients but zero
            assert name in ("dq", "dk") and sk == 1, name
            continue
        assert off(torch.zeros_like(exact), exact, bound) > 1, name
        assert off(2 * exact, exact, bound) > 1 and off(0.95 * exact, exact, bound) > 1, name
        last = exact.clone()
        last[:, -1] = 0
        if (exact[:, -1].norm(dim=-1) > 8 * bound[:, -1]).any():
            assert off(last, exact, bound) > 1, name
        swapped = exact.roll(1, -1)
        assert off(swapped, exact, bound) > 1, name
        other = less_keys if name in ("out", "dq") else less_queries
        if other is not None and not torch.allclose(other[name][0], exact):
            assert off(other[name][0], exact, bound) > 1, name


@pytest.mark.parametrize("dtype,wtype", [(BF16, BF16), (BF16, FP32), (FP16, FP16), (FP16, FP32)])
@pytest.mark.parametrize("kind", [None, "relu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m,k,n", [s for s in SIZES if s[0] * s[1] * s[2] < 10 ** 8])
def test_linear_bounds(dtype, wtype, kind, m, k, n):
    torch.manual_seed(m + k + n)
    x, w, b = rand(m, k, dtype=dtype), rand(n, k, dtype=wtype, std=k ** -0.5), rand(n, dtype=wtype)
    dy = rand(m, n, dtype=dtype)
    rows = linear_rows(x, w, b, None, dy, kind)
    # what the kernels do: the weight in the inputs' type, the slope of the rounded product, rounded
    p = x.double() @ w.to(dtype).double().t() + b.double()
    want = linear64(x, w, b, None, dy, kind)
    g = dy.double() * act64(p.to(dtype).double(), kind)[1] if kind else dy.double()
    gr = g.to(dtype).double()
    as_kernels = {"y": act64(p, kind)[0].to(dtype), "dx": (gr @ w.to(dtype).double()).to(dtype), "dw": (gr.t() @ x.double()).to(wtype),
                  "db": g.sum(0).to(wtype)}
    for name, (exact, bound) in rows.items():
        assert off(as_kernels[name], exact, bound) <= 1, name
        assert off(torch.zeros_like(exact), exact, bound) > 1 and off(2 * exact, exact, bound) > 1, name
        last = exact.clone()
        last[-1] = 0
        assert off(last, exact, bound) > 1 or (exact[-1].norm() <= 8 * bound[-1]), name
        assert torch.equal(exact, want[name][0].reshape(exact.shape))
