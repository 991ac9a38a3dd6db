"""Dropout's kernels against its definition, by themselves, in the layer norm and in attention."""
import pytest
import torch

from _dropout import attention64, kept, kept_count, kept_probabilities
from _layers import U, close, norm64
from hipress_b200.ops import attention, dropout, layer_norm, self_attention

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
SEED = 0x1234567890ABCDEF


def rand(*shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(*shape, device="cuda") * std + mean).to(dtype)


def on_cpu(x, p, seed, site=0, residual=None):
    return dropout(x.cpu(), p, seed=seed, site=site, residual=None if residual is None else residual.cpu())


# ------------------------------------------------------------------ by itself
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("n", [1, 7, 31, 32, 33, 255, 1023, 1024, 1025, 8191, 8192, 8193, 100003])
@pytest.mark.parametrize("p", [0.1, 0.5, 0.99])
def test_dropout(dtype, n, p):
    torch.manual_seed(n)
    x, r, dy = (rand(n, dtype=dtype) for _ in range(3))
    for residual in (None, r):
        leaves = [t.clone().requires_grad_(True) for t in (x, r)]
        y = dropout(leaves[0], p, seed=SEED, site=5, residual=None if residual is None else leaves[1])
        # the same operations in 32 bits, and one rounding: the same bits
        assert torch.equal(y.cpu(), on_cpu(x, p, SEED, 5, residual))
        got = torch.autograd.grad(y, leaves, dy, allow_unused=True)
        assert torch.equal(got[0].cpu(), on_cpu(dy, p, SEED, 5))
        assert got[1] is None if residual is None else torch.equal(got[1], dy)


@pytest.mark.parametrize("seed", [0, -1, 2 ** 63 - 1, -2 ** 63])
@pytest.mark.parametrize("p,site", [(0.25, 0), (0.75, 2 ** 32 - 1), (0.0625, 1), (1e-4, 2), (0.99999, 3)])
def test_seeds_and_probabilities(seed, p, site):
    x = rand(3000, dtype=FP32).abs() + 1
    want = on_cpu(x, p, seed, site)
    for s in (seed, torch.tensor([seed], device="cuda"), torch.tensor(seed, device="cuda")):
        assert torch.equal(dropout(x, p, seed=s, site=site).cpu(), want)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_layouts(dtype):
    torch.manual_seed(0)
    base, more = rand(70, 41, dtype=dtype), rand(70 * 41 + 1, dtype=dtype)
    r = more[1:].view(70, 41)                      # off 16-byte boundaries
    for x, res in ((base.t(), None), (more[1:], None), (base, r), (r, base), (base[::2, 3:], None), (base[:, :1].expand(70, 41), r)):
        assert torch.equal(dropout(x, 0.3, seed=1, residual=res).cpu(), on_cpu(x, 0.3, 1, 0, res))
    leaf = base.clone().requires_grad_(True)
    dropout(leaf, 0.3, seed=1).sum().backward()    # a gradient that is one number, expanded
    assert torch.equal(leaf.grad.cpu(), on_cpu(torch.ones_like(base), 0.3, 1))


def test_dropped_elements_are_zero_whatever_they_are():
    m = kept((4096,), 0.5, 3, 0, "cuda")
    x = torch.where(m, 1.0, float("nan"))
    assert torch.equal(dropout(x, 0.5, seed=3), torch.where(m, 2.0, 0.0))


def test_empty():
    assert dropout(torch.zeros(0, 7, device="cuda"), 0.5, seed=1).shape == (0, 7)
    leaf = torch.zeros(0, 7, device="cuda", requires_grad=True)
    assert torch.autograd.grad(dropout(leaf, 0.5, seed=1).sum(), leaf)[0].shape == (0, 7)


def test_more_than_32_bits_of_elements():
    n = 2 ** 32 + 4096 + 5
    x = torch.ones(n, dtype=BF16, device="cuda")
    y = dropout(x, 0.5, seed=9, site=2)
    from _dropout import kept_bits
    for word in (0, 2 ** 27 - 1, 2 ** 27, 2 ** 27 + 100):
        want = [2.0 if b else 0.0 for b in kept_bits(word, 9, 2, 32768)]
        assert y[32 * word:32 * word + 32].tolist() == want
    assert y[-5:].tolist() == [2.0 if b else 0.0 for b in kept_bits(n // 32, 9, 2, 32768)][:5]


def test_streams_and_repeatability():
    x = rand(1 << 20, dtype=BF16)
    want = dropout(x, 0.1, seed=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [dropout(x, 0.1, seed=4) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, want) for g in got)


def test_captured_steps_move_on_with_their_seed():
    torch.manual_seed(0)
    seed = torch.tensor([100], device="cuda")
    x, w, r, dz = rand(64, 200, dtype=BF16), rand(200, dtype=FP32), rand(64, 200, dtype=BF16), rand(64, 200, dtype=BF16)
    qkv, do = rand(2, 70, 3, 2, 64, dtype=BF16), rand(2, 70, 2, 64, dtype=BF16)

    def step(x, w, r, qkv):
        seed.add_(1)
        s = seed.clone()
        y, z = layer_norm(x, w, residual=dropout(r, 0.2, seed=s), dropout=0.1, seed=s, site=1)
        o = self_attention(qkv, dropout=0.1, seed=s, site=2)
        return [y, z, o, *torch.autograd.grad((y, z, o), (x, w, r, qkv), (dz, dz, do))]

    leaves = lambda: [t.clone().requires_grad_(True) for t in (x, w, r, qkv)]  # noqa: E731
    mine = leaves()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*mine)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*mine)
    seen = []
    for s in (500, 501, 7):
        seed.fill_(s)
        graph.replay()
        seen.append([t.clone() for t in out])
    for s, got in zip((500, 501, 7), seen):
        seed.fill_(s)
        for a, b in zip(got, step(*leaves())):
            assert torch.equal(a, b)
    assert not torch.equal(seen[0][1], seen[1][1])


def test_a_seed_that_moves_between_the_passes_is_refused():
    for call in (lambda x, s: dropout(x, 0.5, seed=s), lambda x, s: layer_norm(x, residual=x, dropout=0.5, seed=s)[1],
                 lambda x, s: self_attention(x.view(2, 4, 3, 1, 8), dropout=0.5, seed=s)):
        seed, x = torch.tensor([4], device="cuda"), rand(8, 24, dtype=BF16).requires_grad_(True)
        y = call(x, seed)
        seed.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_refusals_on_the_gpu():
    x = rand(4, 8, dtype=BF16)
    with pytest.raises(ValueError, match="tensors on"):
        dropout(x, 0.5, seed=torch.tensor([1]))
    with pytest.raises(TypeError):
        dropout(x.double(), 0.5, seed=1)
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(dropout(leaf, 0.5, seed=1).float().square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()
    import torch.autograd.forward_ad as fw
    with fw.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
        dropout(fw.make_dual(x, torch.ones_like(x)), 0.5, seed=1)


# ------------------------------------------------------ in front of a layer norm
def check_norm(x, w, b, r, dy, dz, p, seed, site, dx_roundings=1):
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, w, b, r)]
    y, z = layer_norm(leaves[0], leaves[1], leaves[2], residual=leaves[3], dropout=p, seed=seed, site=site)
    assert torch.equal(z, dropout(x, p, seed=seed, site=site, residual=r))
    want = norm64(z, w, b, dy, dz, 1e-5)
    got = iter(torch.autograd.grad((y, z), [t for t in leaves if t is not None], (dy, dz)))
    grads = {n: next(got) if t is not None else None for n, t in zip("xwbr", leaves)}
    rows, t = x.numel() // x.shape[-1], x.dtype
    steps = 64 + x.shape[-1] // 32
    close(y, *want["y"], 1, t, "y", steps)
    close(grads["r"], *want["dx"], 1, t, "dr", steps)
    m = kept(x.shape, p, seed, site, x.device).double() * (65536 / kept_count(p))
    close(grads["x"], want["dx"][0] * m, want["dx"][1] * m, dx_roundings, t, "dx", steps)
    assert not grads["x"][m == 0].any()
    if w is not None:
        close(grads["w"], *want["dw"], 1, w.dtype, "dw", steps + rows // 8)
    if b is not None:
        close(grads["b"], *want["db"], 1, b.dtype, "db", 64 + rows // 8)


@pytest.mark.parametrize("dtype,wtype", [(BF16, FP32), (FP16, FP16), (FP32, FP32)])
@pytest.mark.parametrize("cols", [8, 9, 33, 200, 257, 513, 769, 1000, 1023, 1024, 1027, 1600, 2047, 2056, 2561, 4095, 4096, 4999,
                                  6144, 8191, 8192, 12001, 16001])
def test_norm_many_rows(dtype, wtype, cols):
    torch.manual_seed(cols)
    rows = min(2051, 8_000_000 // cols)
    x, w, b = rand(rows, cols, dtype=dtype, mean=0.5), rand(cols, dtype=wtype, mean=1), rand(cols, dtype=wtype)
    r, dy, dz = (rand(rows, cols, dtype=dtype) for _ in range(3))
    long = cols > (8192 if dtype == FP32 else 16384) - 8   # one operator after the other, and one rounding more
    check_norm(x, w, b, r, dy, dz, 0.1 if cols % 2 else 0.5, SEED, cols, 2 if long else 1)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 7), (2, 1024), (5, 20000), (4097, 3)])
def test_norm_small_and_long(dtype, rows, cols):
    torch.manual_seed(rows * 7 + cols)
    x, r, dy, dz = (rand(rows, cols, dtype=dtype) for _ in range(4))
    check_norm(x, None, None, r, dy, dz, 0.3, 5, 1, 2)


def test_norm_layouts_and_wanted_gradients():
    torch.manual_seed(3)
    base, w = rand(64, 2 * 136, dtype=BF16), rand(136, dtype=FP32)
    x, r = base[:, :136], base[:, 136:]                       # padded rows
    dy, dz = rand(64, 136, dtype=BF16), rand(136, 64, dtype=BF16).t()
    check_norm(x, w, None, r, dy, dz, 0.2, 1, 1)
    odd = rand(64 * 136 + 1, dtype=BF16)[1:].view(64, 136)     # off 16-byte boundaries
    check_norm(odd, w, None, r, dy, dz, 0.2, 1, 1, 2)
    full = [t.clone().requires_grad_(True) for t in (x, w, r)]
    y, z = layer_norm(full[0], full[1], residual=full[2], dropout=0.2, seed=1, site=1)
    want = dict(zip("xwr", torch.autograd.grad((y, z), full, (dy, dz))))
    for names in ("x", "r", "w", "xw", "wr"):
        some = {n: t.clone().requires_grad_(n in names) for n, t in zip("xwr", (x, w, r))}
        y, z = layer_norm(some["x"], some["w"], residual=some["r"], dropout=0.2, seed=1, site=1)
        outs, gs = ((y, z), (dy, dz)) if names != "w" else ((y,), (dy,))
        for n, g in zip(names, torch.autograd.grad(outs, [some[n] for n in names], gs)):
            assert torch.equal(g, want[n]), (names, n)
    leaf = [x.clone().requires_grad_(True), r.clone().requires_grad_(True)]
    _, z = layer_norm(leaf[0], w, residual=leaf[1], dropout=0.2, seed=1, site=1)   # only the sum is used further on
    dx, dr = torch.autograd.grad(z, leaf, dz)
    assert torch.equal(dr, dz) and torch.equal(dx, dropout(dz, 0.2, seed=1, site=1))


# ------------------------------------------------------------------- attention
def check_attention(b, sq, sk, heads, kv_heads, dim, dtype, causal, lengths, p, seed=SEED, site=3, scale=None):
    torch.manual_seed(sq * 31 + sk)
    q, do = (rand(b, sq, heads, dim, dtype=dtype) for _ in range(2))
    k, v = (rand(b, sk, kv_heads, dim, dtype=dtype) for _ in range(2))
    mask = None
    if lengths is not None:
        mask = torch.arange(sk, device="cuda")[None] < torch.tensor(lengths, device="cuda")[:, None]
        k[~mask], v[~mask] = float("nan"), float("inf")      # what a masked key holds does not matter
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out, lse = attention(*leaves, causal=causal, key_mask=mask, return_lse=True, dropout=p, seed=seed, site=site, scale=scale)
    got = torch.autograd.grad(out, leaves, do)
    m = kept_probabilities(b, heads, sq, sk, p, seed, site, "cuda")
    want = attention64(*(t.detach() for t in leaves), do, causal=causal, mask=mask, kept=m, up=65536 / kept_count(p), scale=scale)
    group = heads // kv_heads
    # p and the result; the result before (delta), ds and the result
    close(out, *want["out"], 2, dtype, "out", 256 + sk // 16)
    rows = want["lse"][0] != -torch.inf
    assert torch.equal(lse != -torch.inf, rows)
    assert (lse[rows] - want["lse"][0][rows]).abs().max() < 1e-4 if rows.any() else True
    close(got[2], *want["dv"], 2, dtype, "dv", 256 + sq * group // 16)
    close(got[0], *want["dq"], 3, dtype, "dq", 256 + sk // 16)
    close(got[1], *want["dk"], 3, dtype, "dk", 256 + sq * group // 16)
    if mask is not None:
        assert not got[1][~mask].any() and not got[2][~mask].any()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("p", [0.1, 0.5, 0.9])
@pytest.mark.parametrize("sq,sk,dim,causal", [(128, 128, 64, False), (128, 128, 64, True), (33, 33, 64, True), (1, 1, 64, False),
                                              (100, 65, 32, False), (31, 127, 64, True), (127, 32, 40, True), (1, 128, 64, False)])
def test_attention_short(dtype, p, sq, sk, dim, causal):
    check_attention(2, sq, sk, 3, 3, dim, dtype, causal, None, p)
    check_attention(2, sq, sk, 3, 3, dim, dtype, causal, [sk, sk // 2], p)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("sq,sk,dim,causal", [(129, 129, 64, True), (200, 333, 64, False), (333, 200, 64, True), (1, 1000, 64, False),
                                              (64, 129, 128, False), (300, 300, 128, True), (517, 1001, 80, False), (1000, 96, 128, True),
                                              (257, 256, 8, False)])
def test_attention_tiles(dtype, sq, sk, dim, causal):
    check_attention(2, sq, sk, 2, 2, dim, dtype, causal, None, 0.1)
    check_attention(2, sq, sk, 2, 2, dim, dtype, causal, [sk, sk // 3], 0.5)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("sq,sk,causal", [(70, 90, False), (300, 300, True), (129, 700, False)])
def test_attention_shared_heads(dim, sq, sk, causal):
    check_attention(3, sq, sk, 8, 2, dim, BF16, causal, None, 0.2)
    check_attention(3, sq, sk, 6, 1, dim, FP16, causal, [sk, 1, sk - 5], 0.2)


def test_attention_two_tiles_a_cta():
    check_attention(4, 700, 400, 16, 16, 128, BF16, False, None, 0.1)
    check_attention(2, 1300, 1300, 16, 4, 128, FP16, True, None, 0.1)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_attention_with_workspaces_full_of_nan(dtype):
    """What the workspaces held before has no effect."""
    for shape in ((2, 1, 1000, 2, 2, 64), (2, 300, 200, 4, 2, 128), (1, 100, 100, 2, 2, 64)):
        junk = [torch.full((1 << k,), float("nan"), device="cuda") for k in range(8, 22) for _ in range(4)]
        del junk
        check_attention(*shape, dtype, False, None, 0.3)


def test_attention_rows_that_see_nothing():
    check_attention(2, 40, 30, 2, 2, 64, BF16, True, [30, 0], 0.3)
    check_attention(2, 400, 150, 2, 1, 64, FP16, True, [150, 0], 0.3)
    check_attention(1, 300, 200, 2, 2, 128, BF16, True, [0], 0.3)


def test_attention_scale_and_seeds():
    check_attention(1, 150, 150, 2, 2, 64, BF16, False, None, 0.1, seed=-1, site=2 ** 32 - 1, scale=-0.2)
    check_attention(1, 90, 90, 2, 2, 64, FP16, False, None, 0.1, seed=2 ** 62, site=0, scale=0.0)


def test_attention_lse_and_kept_results_do_not_depend_on_the_dropout():
    q = rand(2, 200, 3, 4, 64, dtype=BF16)
    a, la = self_attention(q, return_lse=True)
    b, lb = self_attention(q, return_lse=True, dropout=0.3, seed=1)
    c, lc = self_attention(q, return_lse=True, dropout=0.3, seed=1)
    assert torch.equal(la, lb) and torch.equal(b, c) and not torch.equal(a, b)


def test_attention_gradients_are_repeatable():
    q = rand(2, 333, 3, 4, 64, dtype=BF16).requires_grad_(True)
    do = rand(2, 333, 4, 64, dtype=BF16)
    runs = [torch.autograd.grad(self_attention(q, causal=True, dropout=0.1, seed=3), q, do)[0] for _ in range(3)]
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_expected_output_is_that_without_a_dropout(dtype):
    """The mean over seeds: what is kept is scaled by the inverse of its probability."""
    q = rand(1, 64, 3, 1, 64, dtype=dtype)
    want = self_attention(q).double()
    n = 400
    outs = torch.stack([self_attention(q, dropout=0.5, seed=s).double() for s in range(n)])
    sigma = outs.std(0) / n ** 0.5
    # 4096 values: six standard errors, and the roundings of the sums' mean
    assert ((outs.mean(0) - want).abs() <= 6 * sigma + 4 * U[dtype] * want.abs() + 4 * U[dtype]).all()


def test_attention_without_keys_or_queries():
    for sq, sk in ((5, 0), (0, 5), (200, 0)):
        q = rand(2, sq, 4, 64, dtype=BF16).requires_grad_(True)
        k, v = (rand(2, sk, 2, 64, dtype=BF16).requires_grad_(True) for _ in range(2))
        o = attention(q, k, v, dropout=0.5, seed=1)
        assert o.shape == q.shape and not o.any()
        for g in torch.autograd.grad(o, (q, k, v), torch.ones_like(o)):
            assert not g.any()


# ------------------------------------------------------------------ kept tensors
def test_tensors_kept_elsewhere_and_recomputed_passes():
    from torch.utils.checkpoint import checkpoint
    from hipress_b200.ops import cross_entropy
    torch.manual_seed(0)
    x, r, w = rand(40, 3 * 128, dtype=BF16), rand(40, 3 * 128, dtype=BF16), rand(3 * 128, dtype=FP32)
    seed, labels = torch.tensor([12], device="cuda"), torch.randint(0, 128, (40,), device="cuda")

    def step(x, r, w):
        y, z = layer_norm(dropout(x, 0.1, seed=seed, site=1), w, residual=r, dropout=0.2, seed=seed, site=2)
        o = self_attention(y.view(2, 20, 3, 2, 64), dropout=0.3, seed=seed, site=3)
        return cross_entropy(o.reshape(40, 128), labels) + z.float().mean()

    def run(how):
        leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
        loss = how(leaves)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]

    want = run(lambda l: step(*l))
    with torch.autograd.graph.save_on_cpu():
        leaves = [t.clone().requires_grad_(True) for t in (x, r, w)]
        loss = step(*leaves)
    got = [loss.detach(), *torch.autograd.grad(loss, leaves)]
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    again = [t.clone().requires_grad_(True) for t in (x, r, w)]
    loss = checkpoint(step, *again, use_reentrant=False)   # the same masks when the forward pass is run again
    loss.backward()
    assert all(torch.equal(a, b.grad) for a, b in zip(want[1:], again))


# ------------------------------------------------------------------------ BERT
def test_bert_trains_with_all_of_its_dropouts():
    from hipress_b200.models import bert_tiny
    torch.manual_seed(0)
    cpu = bert_tiny(fused="all", seed=5)
    gpu = bert_tiny(fused="all", seed=5).cuda()
    gpu.load_state_dict(cpu.state_dict())
    ids = torch.randint(0, 1000, (3, 40))
    labels = torch.where(torch.rand(3, 40) < 0.3, ids, -100)
    mask = torch.arange(40)[None] < torch.tensor([[40], [17], [31]])
    labels = torch.where(mask, labels, -100)
    want = cpu(ids, labels, key_mask=mask)
    want.backward()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = gpu(ids.cuda(), labels.cuda(), key_mask=mask.cuda())
    got.backward()
    # the same masks on both: what is left is a dozen roundings to bfloat16 in a row
    assert abs(got.item() - want.item()) < 0.02 * abs(want.item())
    for (n, a), b in zip(gpu.named_parameters(), cpu.parameters()):
        if b.grad is not None:
            assert (a.grad.cpu() - b.grad).norm() <= 0.06 * b.grad.norm() + 1e-6, n
    gpu.eval(), cpu.eval()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        p = gpu.score(ids.cuda(), labels.cuda(), key_mask=mask.cuda(), top=4)
    q = cpu.score(ids, labels, key_mask=mask, top=4)
    assert torch.allclose(p.log_probs.cpu(), q.log_probs, atol=0.05) and p.top_tokens.shape == q.top_tokens.shape
