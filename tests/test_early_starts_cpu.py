"""Kernels that start while the one ahead of them still runs (programmatic dependent launch): a bounded wait may only begin once that one
has ended, or its limit runs out over another kernel's work and the product is given up with nothing wrong.  Read from the sources: whether a
limit runs out on a GPU depends on what else it has to do."""
import re
from pathlib import Path

from test_warp_waits_cpu import blocks_of, code_of

CSRC = Path(__file__).resolve().parent.parent / "tiny_llm_infer_b200" / "csrc"
BOUNDED = re.compile(r"\b(?:mbar_wait|warp_wait|quick_wait|finish_tile<[^;]*?>)\(")


def early_waits(text):
    """Lines of bounded waits in a kernel with no wait for the kernel ahead before them in the same role (a branch on the warp)."""
    code = code_of(text)
    blocks, bad = blocks_of(code), []
    kernels = [b for b in blocks if "__global__" in b[2]]
    for start, end, _ in kernels:
        for m in BOUNDED.finditer(code, start, end):
            roles = [b for b in blocks if start < b[0] < m.start() < b[1] and re.search(r"\bwarp\b|else$", b[2])]
            # a wait of the kernel ahead at any depth of the role that encloses this one's, before it
            if not any("TLLM_PDL_WAIT()" in code[b[0]:m.start()] for b in roles):
                bad.append(text.count("\n", 0, m.start()) + 1)
    return bad


def test_bounded_waits_begin_after_the_kernel_ahead():
    text = (CSRC / "fp8_tcgen05.cu").read_text()
    assert "launch_pdl" in text and early_waits(text) == []


def test_the_reading_finds_what_it_looks_for():
    kernel = "__global__ void k() { if (warp == 0) { TLLM_PDL_WAIT(); for (;;) { mbar_wait(&a, 0); } } else { %s if (quick_wait(&a, 0)) return; } }"
    assert early_waits(kernel % "") == [1]
    assert early_waits(kernel % "TLLM_PDL_WAIT();") == []
