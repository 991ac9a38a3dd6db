"""Several devices in one process: what the layer operators settle for each of them."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_what_is_kept_for_each_device(tmp_path):
    exe = tmp_path / "per_device"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", str(ROOT / "csrc/include"), "-o", str(exe),
                    str(ROOT / "tests/native/per_device.cpp")], check=True, timeout=300)
    assert "per device ok" in subprocess.run([str(exe)], capture_output=True, text=True, check=True, timeout=60).stdout


def test_kernel_attributes_are_set_for_each_device():
    """Nothing that a first call finds on its device is kept for the whole process."""
    for name in ("linear.cu", "attention.cu", "layer_norm.cu", "layers_host.cu", "layers.cuh"):
        text = (ROOT / "csrc/cuda" / name).read_text()
        assert not re.search(r"static\s+(const\s+)?(int|cudaError_t)\s+\w+\s*=", text), name
        for m in re.finditer(r"cudaFuncSetAttribute|cudaOccupancyMax", text):
            assert ".get(dev, " in text[max(0, m.start() - 400):m.start()], name


@pytest.mark.multigpu
def test_layers_on_a_second_device():
    from hipress_b200.ops import attention, layer_norm, linear
    torch.manual_seed(0)
    x, w = torch.randn(512, 256, dtype=torch.bfloat16), torch.randn(256, 256, dtype=torch.bfloat16)
    results = []
    for dev in ("cuda:0", "cuda:1"):
        a, b = x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)
        y, z = layer_norm(linear(a, b, activation="gelu"), residual=a)
        o = attention(*(t.view(1, 512, 4, 64) for t in (y, z, y)), causal=True)
        wide = layer_norm(o.reshape(8, 16384).contiguous())
        results.append([t.cpu() for t in (o, wide, *torch.autograd.grad(wide, (a, b), torch.ones_like(wide)))])
    assert all(torch.equal(p, q) for p, q in zip(*results))
