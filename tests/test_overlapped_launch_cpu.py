"""Kernels that start before the one ahead of them has ended read with plain loads.

A read-only load (``__ldg``, or a pointer that is const and __restrict__) promises that
nothing writes the memory while the kernel lives.  These kernels live from before
``wait_for_previous()`` on, while the kernel ahead may still be writing what they read.
"""
import re
from pathlib import Path

CSRC = next(Path(__file__).resolve().parent.parent.glob("minimaxh3*/csrc"))


def _code(path: Path) -> str:
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", path.read_text(), flags=re.S)


def test_no_read_only_loads_where_launches_overlap():
    sources = {p.name: _code(p) for p in CSRC.glob("*.cu*")}
    overlapped = [n for n, s in sources.items() if n.endswith(".cu") and "wait_for_previous()" in s]
    assert {"fp4_quant.cu", "fp4_gemm_sm100.cu", "cross_attention_sm100.cu"} <= set(overlapped)
    for name in overlapped:
        headers = {h for h in re.findall(r'#include "([\w./]+)"', sources[name]) if h in sources}
        for part in {name, *headers}:
            assert not re.search(r"__ldg|__restrict__|ld\.global\.nc", sources[part]), (name, part)
