"""Rules of the layer operators' kernels that no run can show broken: what orders the threads, and
kernels that overlap, stands in their source."""
import re
from pathlib import Path

import pytest

CUDA = Path(__file__).resolve().parent.parent / "csrc" / "cuda"


def kernels(name):
    """Name and body of each kernel of a source file, comments taken out."""
    text = re.sub(r"//[^\n]*", "", (CUDA / name).read_text())
    out = {}
    for m in re.finditer(r"__global__[^{;]*?\b(\w+)\(const __grid_constant__", text):
        start = text.index("{", text.index(")", m.end()))
        depth, at = 1, start + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        out[m.group(1)] = text[start:at]
    return out


@pytest.mark.parametrize("kernel", ["norm_forward_rows", "norm_backward_rows"])
def test_a_slot_is_filled_again_only_behind_its_readers(kernel):
    body = kernels("layer_norm.cu")[kernel]
    loop = body[body.index("ring.wait("):]
    assert loop.count("ring.fetch(") == 1
    reads = [m.start() for m in re.finditer(r"piece\(i, \d\)", loop)]
    assert reads and max(reads) < loop.index("row_sums<NW>(") < loop.index("slot_read<NW>()") < loop.index("ring.fetch(")
    helper = (CUDA / "layer_norm.cu").read_text()
    assert "if (NW == 1) __syncwarp();" in helper[helper.index("void slot_read()"):][:80]


def test_kernels_overlap_only_once_tensor_memory_is_allocated():
    """A CTA of the kernel behind may hold tensor memory while it waits for the one in front: that
    one must not be waiting for room."""
    seen = 0
    for source in ("linear.cu", "attention.cu"):
        for name, body in kernels(source).items():
            if "tmem_alloc<" not in body:
                continue
            seen += 1
            assert body.count("tmem_alloc<") == body.count("dependents_may_start()") == 1, name
            between = body[body.index("tmem_alloc<"):body.index("dependents_may_start()")] \
                if body.index("tmem_alloc<") < body.index("dependents_may_start()") else ""
            assert "__syncthreads();" in between, name
    assert seen == 4


def test_errors_that_are_returned_are_not_left_for_the_next_launch():
    """The runtime keeps the last error for whoever asks: a refused call made the next kernel of
    another library look as if it had failed."""
    for name in ("layers.cuh", "layers_host.cu", "linear.cu", "attention.cu", "layer_norm.cu", "column_sums.cuh"):
        text = re.sub(r"//[^\n]*", "", (CUDA / name).read_text())
        for m in re.finditer(r"\bcuda[A-Z]\w+\(", text):
            if m.group() not in ("cudaGetLastError(",):
                assert text[:m.start()].endswith("told("), (name, m.group())


def test_two_pairs_of_ctas_never_share_an_sm():
    """They allocate tensor memory on two SMs, and could wait for one another there."""
    text = (CUDA / "linear.cu").read_text()
    assert 'static_assert(CG == 1 || kSmem > 114 * 1024' in text
    for name in ("attention.cu", "layer_norm.cu"):
        assert "tmem_alloc<2>" not in (CUDA / name).read_text()
