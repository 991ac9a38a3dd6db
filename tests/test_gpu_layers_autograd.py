"""The layer operators' kernels as autograd uses them: gradients of some inputs only, graphs that
are dropped, saved tensors that come back otherwise, tangents."""
import pytest
import torch

from _layers import close, norm64

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
