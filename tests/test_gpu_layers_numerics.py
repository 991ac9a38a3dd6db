"""The layer operators' kernels value by value, where a norm over the whole result shows nothing:
tails of the activations, infinities that a rounding made, gradients far below one."""
import math

import pytest
import torch

from _layers import U, act64

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def rand(*shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(*shape, device="cuda") * std + mean).to(dtype)


def test_linear_empty_sizes_of_any_shape():
    from hipress_b200.ops import linear
    for lead in ((4,), (2, 3), (0, 3), (2, 0, 1), ()):
        for k, n in ((0, 8), (16, 0), (0, 0)):
            x, w = rand(*lead, k, dtype=BF16).requires_grad_(True), rand(n, k, dtype=BF16).requires_grad_(True)
            b, r = rand(n, dtype=BF16).requires_grad_(True), rand(*lead, n, dtype=BF16).requires_grad_(True)
            y = linear(x, w, b, activation="relu", residual=r)
            assert y.shape == (*lead, n)
            if k == 0:
                assert torch.equal(y, (b.float().clamp(min=0) + r.float()).to(BF16))
            dx, dw, db, dr = torch.autograd.grad(y, (x, w, b, r), torch.ones_like(y))
            assert dx.shape == x.shape and not dx.any() and dw.shape == w.shape and not dw.any()
            assert db.shape == b.shape and torch.equal(dr, torch.ones_like(dr))
