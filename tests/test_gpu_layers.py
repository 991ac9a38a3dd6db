"""The layer operators' kernels against the formulas in 64 bits (tests/_layers.py)."""
import pytest
import torch

from _layers import attention64, close, linear64, norm64

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def rand(*shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(*shape, device="cuda") * std + mean).to(dtype)


# ------------------------------------------------------------------ layer norm
def check_norm(x, w, b, r, dy, dz, eps=1e-5):
    from hipress_b200.ops import layer_norm
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b, r)]
    x1, w1, b1, r1 = leaves
    if r is None:
        y = layer_norm(x1, w1, b1, eps=eps)
        z, outs, gs = x, (y,), (dy,)
    else:
        y, z1 = layer_norm(x1, w1, b1, residual=r1, eps=eps)
        z = (x.float() + r.float()).to(x.dtype)
        assert torch.equal(z1, z)
        outs, gs = (y, z1), (dy, dz)
    want = norm64(z, w, b, dy, None if r is None else dz, eps)
    got = iter(torch.autograd.grad(outs, [t for t in leaves if t is not None], gs))
    grads = {n: next(got) if t is not None else None for n, t in zip("xwbr", leaves)}
    rows, t = x.numel() // x.shape[-1], x.dtype
    steps = 64 + x.shape[-1] // 32
    close(y, *want["y"], 1, t, "y", steps)
    close(grads["x"], *want["dx"], 1, t, "dx", steps)
    if r is not None:
        assert torch.equal(grads["r"], grads["x"])
    if w is not None:
        close(grads["w"], *want["dw"], 1, w.dtype, "dw", steps + rows // 8)
    if b is not None:
        close(grads["b"], *want["db"], 1, b.dtype, "db", 64 + rows // 8)


@pytest.mark.parametrize("dtype,wtype", [(BF16, FP32), (BF16, BF16), (FP16, FP32), (FP16, FP16), (FP32, FP32)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 7), (128, 768), (300, 1024), (77, 1000), (33, 4999), (2, 8193),
                                       (5, 20000), (1000, 64), (4097, 512)])
@pytest.mark.parametrize("residual", [False, True])
def test_layer_norm(dtype, wtype, rows, cols, residual):
    torch.manual_seed(rows * 7 + cols)
    x, w, b = rand(rows, cols, dtype=dtype, mean=0.5), rand(cols, dtype=wtype, mean=1), rand(cols, dtype=wtype)
    r = rand(rows, cols, dtype=dtype) if residual else None
    check_norm(x, w, b, r, rand(rows, cols, dtype=dtype), rand(rows, cols, dtype=dtype))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("cols", [8, 9, 33, 200, 257, 513, 769, 1023, 1027, 1600, 2047, 2056, 2561, 3064, 4095, 4096, 4999,
                                  6143, 6144, 8191, 8192, 12001, 16001, 16384])
def test_layer_norm_many_rows(dtype, cols):
    torch.manual_seed(cols)
    rows = min(4099, 20_000_000 // cols)   # several for every group of warps, and not alike many
    x, w, b = rand(rows, cols, dtype=dtype, mean=0.5), rand(cols, dtype=FP32, mean=1), rand(cols, dtype=FP32)
    check_norm(x, w, b, rand(rows, cols, dtype=dtype), rand(rows, cols, dtype=dtype), rand(rows, cols, dtype=dtype))
    check_norm(x, w, b, None, rand(rows, cols, dtype=dtype), None)


@pytest.mark.parametrize("cols", [64, 1000, 1001, 5000])
def test_layer_norm_strides_and_shapes(cols):
    torch.manual_seed(cols)
    wide = rand(3, 6, 2 * cols, dtype=BF16)
    x, dy, r = wide[:, ::2, :cols], wide[:, 1::2, cols:], wide[:, 1::2, :cols]
    check_norm(x, rand(cols, dtype=FP32), rand(cols, dtype=FP32), None, dy, None)
    check_norm(x, rand(cols, dtype=FP32), rand(cols, dtype=FP32), r, dy, x)
    flat = rand(9 * cols + 64, dtype=FP16)
    for shift in (1, 2, 8):   # every alignment of the rows, of each tensor its own
        a = flat[shift:shift + 4 * cols].view(4, cols)
        c = flat[shift + 5:shift + 5 + 4 * cols].view(4, cols)
        check_norm(a, rand(cols, dtype=FP16), rand(cols + 1, dtype=FP16)[1:], c, a, c)


def test_layer_norm_without_weights_and_of_one_vector():
    torch.manual_seed(0)
    x, dy = rand(5, 129, dtype=BF16), rand(5, 129, dtype=BF16)
    check_norm(x, None, None, None, dy, None)
    check_norm(x, rand(129, dtype=BF16), None, None, dy, None)
    check_norm(x, None, rand(129, dtype=BF16), None, dy, None)
    check_norm(x[0], rand(129, dtype=FP32), rand(129, dtype=FP32), None, dy[0], None)


def test_layer_norm_large_mean_and_constant_rows():
    torch.manual_seed(0)
    # the variance of values near 300 is not lost in the square of their mean
    check_norm(rand(64, 768, dtype=FP32, std=0.01, mean=300), rand(768, dtype=FP32), rand(768, dtype=FP32), None,
               rand(64, 768, dtype=FP32), None)
    from hipress_b200.ops import layer_norm
    b = rand(768, dtype=FP32)
    y = layer_norm(torch.full((4, 768), 3.0, device="cuda", dtype=BF16), rand(768, dtype=FP32), b)
    assert torch.equal(y, b.to(BF16).expand(4, 768))


def test_layer_norm_no_rows_and_only_the_sum_used():
    from hipress_b200.ops import layer_norm
    w = torch.ones(16, device="cuda", requires_grad=True)
    x = torch.zeros(0, 16, device="cuda", dtype=BF16, requires_grad=True)
    y = layer_norm(x, w, None)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert dx.shape == (0, 16) and torch.equal(dw, torch.zeros_like(dw))
    x = rand(4, 16, dtype=BF16).requires_grad_(True)
    _, z = layer_norm(x, w, None, residual=rand(4, 16, dtype=BF16))
    dx, dw = torch.autograd.grad(z, (x, w), torch.ones_like(z))
    assert torch.equal(dx, torch.ones_like(dx)) and torch.equal(dw, torch.zeros_like(dw))


def test_layer_norm_gradient_against_differences():
    from hipress_b200.ops import layer_norm
    torch.manual_seed(3)
    x, w, b = rand(6, 96, dtype=FP32), rand(96, dtype=FP32), rand(96, dtype=FP32)
    dy, t = rand(6, 96, dtype=FP32), rand(6, 96, dtype=FP32)
    x1 = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(layer_norm(x1, w, b), x1, dy)
    step = 2.0 ** -7
    value = lambda s: (layer_norm(x + s * step * t, w, b).double() * dy.double()).sum()  # noqa: E731
    slope = (value(1) - value(-1)) / (2 * step)
    # third order: about step^2 of the slope's scale; 32-bit values: 2^-24 / step
    assert abs(slope - (dx.double() * t.double()).sum()) <= 24 * (step ** 2 + 2.0 ** -24 / step) * 24


# ---------------------------------------------------------------------- linear
def check_linear(x, w, b, r, dy, kind):
    from hipress_b200.ops import linear
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b, r)]
    y = linear(leaves[0], leaves[1], leaves[2], activation=kind, residual=leaves[3])
    got = iter(torch.autograd.grad(y, [t for t in leaves if t is not None], dy))
    dx, dw, db, dr = (next(got) if t is not None else None for t in leaves)
    want = linear64(x, w, b, r, dy, kind)
    t, k, m, n = x.dtype, x.shape[-1], x.numel() // max(1, x.shape[-1]), w.shape[0]
    cast = 1 if w.dtype != t else 0     # the weight's own rounding
    early = 2 if kind else 0            # the product's, whose slope is taken, and the slope's result's
    close(y.reshape(-1, n), *want["y"], 1 + cast, t, "y", 64 + k // 16)
    close(dx.reshape(-1, k), *want["dx"], 1 + cast + early, t, "dx", 64 + n // 16)
    for name, g, wt in (("dw", dw, w.dtype), ("db", db, b.dtype if b is not None else None)):
        if g is None:
            continue
        if wt == FP32 and not early:    # sums of exact products
            close(g, *want[name], 0, t, name, 64 + m // 16)
        else:
            close(g, *want[name], 1 + early + cast, t, name, 64 + m // 16)
    if r is not None:
        assert torch.equal(dr, dy)
    y2 = linear(x, w, b, activation=kind, residual=r)
    assert torch.equal(y2, y), "with and without a gradient"


SIZES = [(1, 8, 8), (1, 1, 1), (5, 3, 7), (33, 512, 2048), (128, 768, 768), (129, 257, 300), (257, 64, 1000), (640, 1024, 520),
         (1000, 136, 8), (7, 2050, 31), (300, 40, 1025), (2100, 72, 264)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("kind", [None, "relu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear(dtype, kind, m, k, n):
    torch.manual_seed(m + k + n)
    for wtype, residual in ((dtype, False), (FP32, True)):
        x, w, b = rand(m, k, dtype=dtype), rand(n, k, dtype=wtype, std=k ** -0.5), rand(n, dtype=wtype)
        check_linear(x, w, b, rand(m, n, dtype=dtype) if residual else None, rand(m, n, dtype=dtype), kind)


def test_linear_strides():
    torch.manual_seed(1)
    for cols, shift in ((256, 0), (256, 8), (250, 3), (64, 1)):
        wide = rand(100, 1024, dtype=BF16)
        x, dy, r = wide[:, shift:shift + cols], wide[:, 300 + shift:300 + shift + 200], wide[:, 511:711]
        w = rand(200, cols + 24, dtype=BF16, std=0.1)[:, 8:8 + cols]
        check_linear(x, w, rand(200, dtype=BF16), r, dy, "gelu")
        check_linear(x, rand(cols, 200, dtype=BF16, std=0.1).t(), None, None, dy, None)
    x = rand(4, 6, 32, dtype=FP16).transpose(0, 1)
    check_linear(x, rand(48, 32, dtype=FP16), None, None, rand(6, 4, 48, dtype=FP16), None)
    check_linear(x[0, 0], rand(48, 32, dtype=FP16), None, None, rand(48, dtype=FP16), "relu")
    dy = rand(1, 48, dtype=FP16).expand(24, 48)    # the gradient of a sum over rows
    check_linear(rand(24, 32, dtype=FP16), rand(48, 32, dtype=FP16), rand(48, dtype=FP16), None, dy, None)


def test_linear_empty_sizes():
    from hipress_b200.ops import linear
    for m, k, n in ((0, 16, 8), (4, 0, 8), (4, 16, 0)):
        x, w = rand(m, k, dtype=BF16).requires_grad_(True), rand(n, k, dtype=BF16).requires_grad_(True)
        b = rand(n, dtype=BF16).requires_grad_(True)
        y = linear(x, w, b, activation="relu")
        assert y.shape == (m, n)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
        assert dx.shape == x.shape and not dw.any() and torch.equal(y, b.clamp(min=0).expand(m, n)) or k == 16
        if m == 0:
            assert not dw.any() and not db.any()
        if n == 0:
            assert not dx.any()


def test_linear_keeps_infinities_and_nan_in_their_rows():
    from hipress_b200.ops import linear
    torch.manual_seed(2)
    x, w = rand(200, 128, dtype=BF16), rand(300, 128, dtype=BF16)
    clean = linear(x, w)
    x[3, 5], x[77, 0] = float("nan"), float("inf")
    y = linear(x, w)
    assert torch.isnan(y[3]).all() and not torch.isfinite(y[77]).any()
    rest = [i for i in range(200) if i not in (3, 77)]
    assert torch.equal(y[rest], clean[rest])


# ------------------------------------------------------------------- attention
def check_attention(q, k, v, do, *, causal=False, mask=None, scale=None):
    from hipress_b200.ops import attention
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out, lse = attention(*leaves, causal=causal, key_mask=mask, scale=scale, return_lse=True)
    dq, dk, dv = torch.autograd.grad(out, leaves, do)
    want = attention64(q, k, v, do, causal=causal, mask=mask, scale=scale)
    t, sq, sk, group = q.dtype, q.shape[1], k.shape[1], q.shape[2] // k.shape[2]
    seen = torch.isfinite(want["lse"][0])
    assert torch.equal(torch.isfinite(lse), seen)
    s = 1 + want["lse"][0][seen].abs().amax() if seen.any() else torch.tensor(1.0)
    assert (lse[seen].double() - want["lse"][0][seen]).abs().amax() <= 2.0 ** -18 * s if seen.any() else True
    # an exponent's error, 2^-18 of a few units, counts like so many additions
    close(out, *want["out"], 2, t, "out", 256 + sk // 16)                # p and the result
    close(dv, *want["dv"], 2, t, "dv", 256 + sq * group // 16)
    close(dq, *want["dq"], 3, t, "dq", 256 + sk // 16)                   # the result before, ds and the result
    close(dk, *want["dk"], 3, t, "dk", 256 + sq * group // 16)
    nothing = ~seen.transpose(1, 2)
    assert not out[nothing].any() and not dq[nothing].any()
    if mask is not None:
        assert not dk[~mask].any() and not dv[~mask].any()
    o2, l2 = attention(q, k, v, causal=causal, key_mask=mask, scale=scale, return_lse=True)
    assert torch.equal(o2, out) and torch.equal(l2, lse)
    again = torch.autograd.grad(attention(*leaves, causal=causal, key_mask=mask, scale=scale), leaves, do)
    assert all(torch.equal(x, y) for x, y in zip(again, (dq, dk, dv))), "the same call twice"


SHAPES = [  # batch, queries, keys, heads, key heads, dim
    (1, 1, 1, 1, 1, 8), (2, 33, 33, 8, 8, 64), (3, 1, 300, 4, 2, 64), (2, 128, 128, 3, 3, 64), (1, 129, 257, 4, 1, 128),
    (2, 300, 70, 2, 2, 40), (1, 64, 1000, 6, 3, 72), (1, 1000, 64, 2, 1, 16), (5, 17, 19, 2, 2, 120), (1, 513, 513, 2, 2, 128),
    (1, 700, 700, 1, 1, 64), (70, 5, 7, 2, 2, 32), (1, 2, 129, 1, 1, 128)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("masked", [None, "lengths", "holes"])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(dtype, causal, masked, shape):
    b, sq, sk, h, hk, d = shape
    torch.manual_seed(sq + sk + d)
    q, do = rand(b, sq, h, d, dtype=dtype), rand(b, sq, h, d, dtype=dtype)
    k, v = rand(b, sk, hk, d, dtype=dtype), rand(b, sk, hk, d, dtype=dtype)
    mask = None
    if masked == "lengths":
        mask = torch.arange(sk, device="cuda")[None] < torch.randint(0, sk + 1, (b, 1), device="cuda")
        mask[0] = False            # a sequence of which nothing is left
    elif masked == "holes":
        mask = torch.rand(b, sk, device="cuda") < 0.6
    check_attention(q, k, v, do, causal=causal, mask=mask)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -65504.0])
def test_attention_masked_keys_hold_anything(dtype, value):
    torch.manual_seed(5)
    b, s, h, d = 2, 200, 2, 64
    q, do = rand(b, s, h, d, dtype=dtype), rand(b, s, h, d, dtype=dtype)
    k, v = rand(b, s, h, d, dtype=dtype), rand(b, s, h, d, dtype=dtype)
    mask = torch.rand(b, s, device="cuda") < 0.7
    mask[1, 128:] = False
    k[~mask], v[~mask] = value, value
    check_attention(q, k, v, do, mask=mask)
    check_attention(q, k, v, do, mask=mask, causal=True)


# more tiles of queries than the SMs hold one by one
MANY = [(8, 300, 70, 16, 16, 40), (5, 257, 400, 24, 8, 64), (3, 700, 700, 20, 20, 64), (1, 400, 1, 80, 1, 8),
        (2, 520, 129, 16, 16, 128), (3, 130, 300, 32, 8, 72)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("masked", [None, "lengths", "holes"])
@pytest.mark.parametrize("shape", MANY)
def test_attention_many_queries(dtype, causal, masked, shape):
    test_attention(dtype, causal, masked, shape)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -65504.0])
def test_attention_many_queries_masked_keys_hold_anything(dim, value):
    torch.manual_seed(12)
    b, s, h = 3, 290, 40
    q, do, k, v = (rand(b, s, h, dim, dtype=BF16) for _ in range(4))
    mask = torch.rand(b, s, device="cuda") < 0.7
    mask[1, 64:] = False
    mask[2] = False
    k[~mask], v[~mask] = value, value
    check_attention(q, k, v, do, mask=mask)
    check_attention(q, k, v, do, mask=mask, causal=True, scale=-0.2)


def test_attention_strides():
    torch.manual_seed(6)
    b, s, h, d = 2, 150, 4, 64
    do = rand(b, s, h, d, dtype=BF16)
    check_attention(*rand(b, s, 3, h, d, dtype=BF16).unbind(2), do)
    check_attention(*(rand(b, h, s, d, dtype=BF16).transpose(1, 2) for _ in range(3)),
                    rand(b, h, s, d, dtype=BF16).transpose(1, 2), causal=True)
    odd = rand(b, s, h, 3 * d + 1, dtype=BF16)     # rows that no tile copy can start at
    check_attention(odd[..., :d], odd[..., d:2 * d], odd[..., 2 * d:3 * d], odd[..., 1:d + 1])
    check_attention(rand(1, s, h, d, dtype=BF16).expand(b, s, h, d), rand(b, s, 1, d, dtype=BF16).expand(b, s, h, d),
                    rand(b, s, h, d, dtype=BF16), rand(b, 1, h, d, dtype=BF16).expand(b, s, h, d))
    mask = (torch.rand(s, b, device="cuda") < 0.7).t()
    check_attention(*rand(b, s, 3, h, d, dtype=BF16).unbind(2), do, mask=mask)
    check_attention(*rand(b, s, 3, h, d, dtype=BF16).unbind(2), do,
                    mask=(torch.rand(b, 2 * s, device="cuda") < 0.7)[:, 3:s + 3])


def test_attention_scales_and_large_scores():
    torch.manual_seed(7)
    q, k, v, do = (rand(1, 140, 2, 64, dtype=FP16) for _ in range(4))
    check_attention(q, k, v, do, scale=0.0)
    check_attention(q, k, v, do, scale=-0.3)
    check_attention(8 * q, 8 * k, v, do, causal=True)    # one key takes nearly everything


def test_attention_empty_sizes():
    from hipress_b200.ops import attention
    for b, sq, sk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q = rand(b, sq, 2, 64, dtype=BF16).requires_grad_(True)
        k, v = (rand(b, sk, 2, 64, dtype=BF16).requires_grad_(True) for _ in range(2))
        o, lse = attention(q, k, v, return_lse=True)
        assert o.shape == q.shape and not o.any() and (lse == -float("inf")).all()
        for g, x in zip(torch.autograd.grad(o, (q, k, v), torch.ones_like(o)), (q, k, v)):
            assert g.shape == x.shape and not g.any()


@pytest.mark.parametrize("causal", [False, True])
def test_self_attention_is_attention(causal):
    from hipress_b200.ops import attention, self_attention
    torch.manual_seed(8)
    qkv = rand(2, 190, 3, 4, 64, dtype=BF16).requires_grad_(True)
    do = rand(2, 190, 4, 64, dtype=BF16)
    mask = torch.rand(2, 190, device="cuda") < 0.8
    o = self_attention(qkv, causal=causal, key_mask=mask)
    g, = torch.autograd.grad(o, qkv, do)
    q, k, v = (t.detach().requires_grad_(True) for t in qkv.unbind(2))
    o2 = attention(q, k, v, causal=causal, key_mask=mask)
    assert torch.equal(o, o2)
    assert torch.equal(g, torch.stack(torch.autograd.grad(o2, (q, k, v), do), 2))


# --------------------------------------------------- streams, autocast, refusals
def test_layers_on_a_stream_of_their_own():
    from hipress_b200.ops import attention, layer_norm, linear
    torch.manual_seed(9)
    x, w, r = rand(300, 256, dtype=BF16), rand(256, 256, dtype=BF16), rand(300, 256, dtype=BF16)

    def chain():
        y, z = layer_norm(linear(x, w, None, activation="gelu"), residual=r)
        return attention(*(t.view(1, 300, 4, 64) for t in (y, z, y))), z

    want = chain()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = chain()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_layers_in_a_thread_that_has_not_used_the_gpu():
    import threading
    from hipress_b200.ops import attention, linear
    torch.manual_seed(11)
    x, w = rand(40, 64, dtype=BF16), rand(64, 64, dtype=BF16)
    want = linear(x, w), attention(*(x.view(1, 40, 1, 64),) * 3)
    got = []
    for call in (lambda: linear(x, w), lambda: attention(*(x.view(1, 40, 1, 64),) * 3)):
        t = threading.Thread(target=lambda: got.append(call()))
        t.start()
        t.join()
    assert len(got) == 2 and all(torch.equal(a, b) for a, b in zip(got, want))


def test_layers_in_a_graph():
    from hipress_b200.ops import attention, layer_norm, linear
    torch.manual_seed(10)
    x, w = rand(200, 256, dtype=BF16), rand(256, 256, dtype=BF16)

    def chain():
        y = layer_norm(linear(x, w, None, activation="gelu"))
        return attention(*(y.view(1, 200, 4, 64) for _ in range(3)), causal=True)

    chain()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain()
    x.copy_(rand(200, 256, dtype=BF16))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, chain())
    del graph


def test_layers_under_autocast():
    from hipress_b200.ops import attention, layer_norm, linear
    x, w = rand(4, 64, dtype=FP32), rand(64, 64, dtype=FP32)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert linear(x, w).dtype == BF16 and torch.equal(linear(x, w), linear(x.to(BF16), w))
        assert attention(*(x.view(1, 4, 1, 64),) * 3).dtype == BF16
        assert layer_norm(x).dtype == FP32


def test_layers_refuse():
    from hipress_b200.ops import attention, linear, self_attention
    x = rand(4, 64, dtype=FP32)
    with pytest.raises(TypeError, match="autocast"):
        linear(x, x)
    with pytest.raises(TypeError, match="autocast"):
        attention(*(x.view(1, 4, 1, 64),) * 3)
    h = x.to(BF16)
    with pytest.raises(ValueError, match="multiple of 8"):
        attention(*(h[:, :60].reshape(1, 4, 1, 60),) * 3)
    with pytest.raises(ValueError, match="multiple of 8"):
        attention(*(rand(1, 4, 1, 136, dtype=BF16),) * 3)
    with pytest.raises(ValueError, match="tensors on"):
        linear(h, h.cpu())
    with pytest.raises(TypeError):
        linear(h, h.half())
    with pytest.raises(ValueError, match="packed|batch, length, 3"):
        self_attention(h)
