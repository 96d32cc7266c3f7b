"""Kernels launched so that they may start before the kernel ahead of them has ended
(harp_b200/csrc/dependent_launch.cuh) read what that kernel wrote: every one of them
waits first, and none reads through the read-only path or by a load that the compiler
may move ahead of the wait.  No run shows such a load to be wrong reliably, so the
sources themselves are looked at."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "harp_b200", "csrc")


def _code(path):
    s = re.sub(r"/\*.*?\*/", " ", open(path).read(), flags=re.S)
    return re.sub(r"//[^\n]*", " ", s)


def _files():
    return [p for p in sorted(glob.glob(os.path.join(CSRC, "*.cu"))) if "launch_dependent(" in _code(p)]


def test_there_are_dependent_launches():
    assert {os.path.basename(p) for p in _files()} >= {"quant.cu", "gemm_s8_sm100.cu"}


@pytest.mark.parametrize("path", _files(), ids=os.path.basename)
def test_loads_are_coherent_and_behind_the_wait(path):
    code = _code(path)
    assert not re.findall(r"__ld(?:g|ca|cg|cs|lu|cv)\b|ld\.global\.nc|__restrict__", code)
    for asm in re.finditer(r"\basm\b(\s+volatile)?\s*\(([^;]*);", code):
        if re.search(r'"\s*ld\.', asm.group(0)):
            assert asm.group(1), asm.group(0)


@pytest.mark.parametrize("path", _files(), ids=os.path.basename)
def test_every_kernel_waits(path):
    code = _code(path)
    starts = [m.start() for m in re.finditer(r"__global__", code)]
    assert starts
    for a in starts:
        body = code[code.index("{", a):]
        depth, end = 0, 0
        for i, c in enumerate(body):
            depth += (c == "{") - (c == "}")
            if depth == 0:
                end = i
                break
        assert "dependency_wait();" in body[:end], code[a:a + 200]
