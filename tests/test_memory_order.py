"""Loads of data that a launch writes itself, read from the sources.

The read-only path (``__ldg``, ``ld.global.nc``) is defined only for memory that nothing writes while
the kernel runs: neither a grid barrier nor a programmatic launch's wait orders it. A stale value
cannot be made to appear at will, so the kernels' sources are checked instead of their outputs.
"""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "cuda-kernel_b200" / "csrc"


def body(text, name):
    """The braces of the function whose definition starts with `name(`."""
    at = next(m.start() for m in re.finditer(rf"\b{name}\(", text) if "{" in text[m.start():].split(";")[0])
    start = text.index("{", at)
    depth = 0
    for i in range(start, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return text[start:i + 1]
    raise AssertionError(name)


def read_only_helpers(text):
    """Functions of the file that reach a non-coherent load whatever their template arguments."""
    names = set(re.findall(r"(?:uint32_t|uint4)\s+(\w+)\(const unsigned char\* row", text))
    return {n for n in names if "__ldg" in body(text, n) and "WRITTEN" not in body(text, n)}


def test_prepared_tokens_are_read_coherently():
    """Their scales lie in the workspace: written by other CTAs of the gate kernel, or by the gate
    kernel while the down kernel is already resident."""
    wide = (CSRC / "wide.cuh").read_text()
    bring = body(wide, "bring")
    assert "__ldg" not in bring and ".nc" not in bring
    for helper in read_only_helpers(wide) | read_only_helpers((CSRC / "tcgen05.cuh").read_text()):
        assert not re.search(rf"\b{helper}\b", bring), helper
    assert set(re.findall(r"scale_word<(\w+)>", bring)) == {"true"}
    # the weights' scales are read-only for the whole launch and keep the cached path
    assert set(re.findall(r"scale_word<(\w+)>", body(wide, "spread"))) == {"false"}


def test_workspace_reads_of_the_layer():
    """The layer's own files read no pointer into the workspace through the read-only path."""
    for name in ("moe.cuh", "moe_wide.cu"):
        text = (CSRC / name).read_text()
        assert "__ldg" not in text and "global.nc" not in text, name
