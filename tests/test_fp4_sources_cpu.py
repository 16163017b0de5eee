"""What can be shown from the 4-bit kernels' sources without a GPU."""

from __future__ import annotations

import re

import pytest

from deterministic_inference_b200.kernels.build import CSRC
from tests.test_kernel_sources_cpu import _braced

SOURCES = ("gemm_fp4.cu", "attention_fp4_stream.cu")


def _kernels(name):
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    for m in re.finditer(r"__global__[^{;]*?(\w+_kernel)\(", text):
        a, b = _braced(text, text.index(") {", m.end()))
        yield m.group(1), text[a:b]


@pytest.mark.parametrize("name", SOURCES)
def test_the_next_kernel_is_let_in_when_tensor_memory_is_taken(name):
    """A block lets the kernel that follows start only behind a barrier behind its allocation of tensor memory: the follower's blocks, which
    wait for this grid's end, could otherwise take what a block of this grid still waits for."""
    found = 0
    for kernel, body in _kernels(name):
        if "tcgen05.alloc" not in body:
            continue
        found += 1
        taken = max(m.start() for m in re.finditer(r"tcgen05\.alloc", body))
        barrier = body.index("__syncthreads()", taken)
        triggers = [m.start() for m in re.finditer(r"pdl_trigger\(|pdl_prologue\(", body)]
        assert triggers and min(triggers) > barrier, f"{name}: {kernel}"
    assert found == (2 if name == "gemm_fp4.cu" else 1)


def test_every_exported_function_is_called():
    """What a 4-bit library exports is called by the package (or by another of its libraries, by address)."""
    package = "".join(p.read_text() for p in (CSRC.parent / "kernels").glob("*.py"))
    for name in ("rows_fp4.cu", "cache_fp4.cu", "gemm_fp4.cu", "attention_fp4.cu", "attention_fp4_stream.cu"):
        text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
        exported = re.findall(r"^(?:int|void) (dib_\w+)\(", text[text.index('extern "C"'):], re.M)
        assert exported
        for f in exported:
            assert re.search(rf"\b{f}\b", package), f"{name}: nobody calls {f}"


def test_pages_made_for_prompts_are_those_the_host_lists():
    from deterministic_inference_b200.kernels import fp4
    text = (CSRC / "cache_fp4.cu").read_text()
    assert int(re.search(r"UNPACK_PAGE = (\d+);", text).group(1)) == fp4.PAGE
