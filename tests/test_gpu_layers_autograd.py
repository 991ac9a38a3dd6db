"""The layer operators' kernels as autograd uses them: gradients of some inputs only, graphs that
are dropped, saved tensors that come back otherwise, tangents."""
import pytest
import torch

from _layers import close, norm64
from test_layers_cpu_edges import OPERATORS, check_second_derivatives

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def rand(*shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(*shape, device="cuda") * std + mean).to(dtype)


def padded(rows, cols, pitch, dtype):
    """Rows on 16-byte boundaries whatever their length; nothing of what is between them may count."""
    wide = torch.full((rows, pitch), float("nan"), device="cuda", dtype=dtype)
    wide[:, :cols] = rand(rows, cols, dtype=dtype, mean=0.5)
    return wide[:, :cols]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows", [1, 2, 41, 1000])
@pytest.mark.parametrize("cols", [9, 70, 500, 1001, 1023, 1500, 3065, 4999, 8191])
def test_layer_norm_weights_gradient_alone_of_padded_rows(dtype, rows, cols):
    from hipress_b200.ops import layer_norm
    torch.manual_seed(rows + cols)
    pitch = (cols + 7) // 8 * 8 + 8
    x, dy = padded(rows, cols, pitch, dtype), padded(rows, cols, pitch, dtype)
    w, b = rand(cols, dtype=FP32, mean=1).requires_grad_(True), rand(cols, dtype=FP32).requires_grad_(True)
    dw, db = torch.autograd.grad(layer_norm(x, w, b), (w, b), dy)
    want = norm64(x, w.detach(), b.detach(), dy, None, 1e-5)
    # each value by itself: what strays from the end of a row does so into a few columns
    for name, got in (("dw", dw), ("db", db)):
        exact, scale = want[name]
        assert ((got.double() - exact).abs() <= (64 + cols // 32 + rows // 8) * 2.0 ** -23 * scale + 1e-30).all(), name
        close(got, exact, scale, 0, FP32, name, 64 + cols // 32 + rows // 8)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("cols", [256, 777, 1024])
def test_layer_norm_rows_of_one_warp_keep_their_third_tensor(dtype, cols):
    """The gradient that goes past the norm is read from the ring and in no sum."""
    from hipress_b200.ops import layer_norm
    torch.manual_seed(cols)
    rows = 40000
    x = rand(rows, cols, dtype=dtype).requires_grad_(True)
    r = torch.zeros_like(x, requires_grad=False)
    dz = (torch.arange(rows, device="cuda") % 97)[:, None].to(dtype).expand(rows, cols).contiguous()
    y, z = layer_norm(x, residual=r)
    # no gradient of y: what arrives is the third tensor
    dx, = torch.autograd.grad((y, z), x, (torch.zeros_like(y), dz))
    assert torch.equal(dx, dz)


def calls():
    """Each operator with everything it keeps for its backward pass: name, call, leaves, odd sizes."""
    from hipress_b200.ops import attention, layer_norm, linear, self_attention
    torch.manual_seed(4)
    g = lambda *s, dtype=BF16, std=1.0: rand(*s, dtype=dtype, std=std).requires_grad_(True)  # noqa: E731
    x, r, nw, nb = g(300, 500), g(300, 500), g(500, dtype=FP32), g(500, dtype=FP32)
    lx, lw, lb, lr = g(3, 70, 131), g(77, 131, std=0.1), g(77), g(3, 70, 77)
    q, k, v, qkv = g(2, 150, 4, 40), g(2, 170, 2, 40), g(2, 170, 2, 40), g(2, 100, 3, 2, 64)
    mask = torch.rand(2, 170, device="cuda") < 0.8
    return {"layer_norm": (lambda: layer_norm(x, nw, nb), (x, nw, nb)),
            "layer_norm residual": (lambda: layer_norm(x, nw, nb, residual=r), (x, nw, nb, r)),
            "linear": (lambda: linear(lx, lw, lb), (lx, lw, lb)),
            "linear gelu": (lambda: linear(lx, lw, lb, activation="gelu", residual=lr), (lx, lw, lb, lr)),
            "attention": (lambda: attention(q, k, v, key_mask=mask), (q, k, v)),
            "attention lse": (lambda: attention(q, k, v, causal=True, return_lse=True)[0], (q, k, v)),
            "self_attention": (lambda: self_attention(qkv), (qkv,))}


NAMES = ["layer_norm", "layer_norm residual", "linear", "linear gelu", "attention", "attention lse", "self_attention"]


@pytest.mark.parametrize("name", NAMES)
def test_a_graph_that_is_dropped_is_freed(name):
    call, _ = calls()[name]
    call()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(5):
        call()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before


def gradients(call, leaves):
    out = call()
    out = out if isinstance(out, tuple) else (out,)
    torch.manual_seed(6)
    return torch.autograd.grad(out, leaves, [rand(*o.shape, dtype=o.dtype) for o in out])


@pytest.mark.parametrize("name", NAMES)
def test_saved_tensors_may_be_kept_elsewhere(name):
    """Offloading brings back what was saved in strides of its own."""
    call, leaves = calls()[name]
    want = gradients(call, leaves)
    with torch.autograd.graph.save_on_cpu():
        got = gradients(call, leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    def wide(t):   # the same values, a column apart, off every boundary
        if t.dim() < 2:
            return t.clone()
        out = torch.empty(*t.shape[:-1], 2 * t.shape[-1] + 1, dtype=t.dtype, device=t.device)[..., 1::2]
        return out.copy_(t)

    with torch.autograd.graph.saved_tensors_hooks(wide, lambda t: t):
        got = gradients(call, leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("change", [lambda t: t.cpu(), lambda t: t.double() if t.is_floating_point() else t.int(), lambda t: t[..., :-1]])
def test_saved_tensors_that_are_others_are_refused(name, change):
    """Another device, type or size than what was saved."""
    call, leaves = calls()[name]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change), pytest.raises(RuntimeError, match="saved tensor"):
        gradients(call, leaves)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode_is_refused(name, leaf):
    import torch.autograd.forward_ad as fwd
    from hipress_b200.ops import attention, layer_norm, linear, self_attention
    torch.manual_seed(5)
    op = {"layer_norm": lambda x: layer_norm(x), "layer_norm residual": lambda x: layer_norm(x.detach(), residual=x),
          "linear": lambda x: linear(x, x.detach()), "linear gelu": lambda x: linear(x.detach(), x, activation="gelu"),
          "attention": lambda x: attention(*(x.view(1, 64, 1, 64),) * 3),
          "attention lse": lambda x: attention(*(x.detach().view(1, 64, 1, 64),) * 2, x.view(1, 64, 1, 64), return_lse=True),
          "self_attention": lambda x: self_attention(x.view(1, 64, 1, 1, 64).expand(1, 64, 3, 1, 64))}[name]
    x, t = rand(64, 64, dtype=BF16), rand(64, 64, dtype=BF16)
    op(x)
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward mode"):
        op(fwd.make_dual(x.requires_grad_(leaf), t))


def test_a_wait_that_ran_out_is_reported_by_the_next_call():
    from hipress_b200._native import lib
    from hipress_b200.ops import linear
    x = rand(8, 16, dtype=BF16)
    want = linear(x, x)
    took = torch.zeros(2, dtype=torch.int64, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.cuda().hp_cuda_layer_wait_probe(50_000_000, took.data_ptr(), stream) == 0
    torch.cuda.synchronize()
    own, beside = took.tolist()
    assert 50_000_000 <= own < 1_000_000_000 and 0 < beside < 1_000_000_000
    with pytest.raises(RuntimeError, match="gave up waiting"):
        linear(x, x)
    assert torch.equal(linear(x, x), want)    # said once; the device is usable


@pytest.mark.parametrize("name", OPERATORS)
def test_second_derivatives_are_refused(name):
    check_second_derivatives("cuda", BF16, name)
