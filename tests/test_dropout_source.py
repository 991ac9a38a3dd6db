"""Rules of the kernels of dropout and log probabilities that no run can show broken (as
tests/test_layers_source.py has them for the other layer operators)."""
import re

from test_layers_source import CUDA, kernels

FILES = ("dropout.cu", "log_probs.cu", "philox.cuh", "layer_norm_dropout.cu")


def test_errors_that_are_returned_are_not_left_for_the_next_launch():
    for name in FILES:
        text = re.sub(r"//[^\n]*", "", (CUDA / name).read_text())
        for m in re.finditer(r"\bcuda[A-Z]\w+\(", text):
            assert text[:m.start()].endswith("told("), (name, m.group())


def test_kernels_touch_memory_only_behind_the_kernel_in_front():
    """Those that may start early wait before they read or write what another kernel may still hold."""
    seen = 0
    for name in FILES:
        for kernel, body in kernels(name).items():
            seen += 1
            assert body.count("wait_for_kernel_before();") == 1, kernel
            before = body[:body.index("wait_for_kernel_before();")]
            assert not re.search(r"\ba\.(x|y|residual|logits|tokens|stats|workspace)\b\s*[\[+]|drop_key\(|row_at\(", before), kernel
    assert seen == 3


def test_copies_ahead_are_read_behind_a_wait_and_overwritten_behind_the_read():
    body = kernels("log_probs.cu")["log_probs_kernel"]
    loop = body[body.index("float top[kBatch];"):]
    wait, read, use, fetch = (loop.index(s) for s in ("cp.async.wait_group", "slot[i * kThreads]", "if (now > sum.m + 8.f", "fetch();"))
    assert wait < read < use < fetch
    assert loop[:loop.index("of_warp(")].count("fetch();") == 1
