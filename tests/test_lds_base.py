"""Kernels that load into LDS by an address of their own making (m0) have one LDS array, which then lies at address 0, or
take the array's address into account."""
from __future__ import annotations

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "osp-next_amd", "csrc")


def kernels(text):
    """(name, body) of the __global__ functions of a source text."""
    for m in re.finditer(r"__global__", text):
        at = text.index("{", text.index(")", text.index("k_", m.end())))
        depth, end = 1, at + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield re.search(r"\bk_\w+", text[m.end():]).group(0), text[at:end]


@pytest.mark.parametrize("name", ["hif8_fp8_gemm.hip", "hif8_gemm_dtl.hip", "hif8_gemm_small.hip"])
def test_one_lds_array(name):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    assert "m0" in text and " lds" in text
    seen = 0
    for kernel, body in kernels(text):
        arrays = re.findall(r"__shared__[^;]*?(\w+)\[", body)
        if "smem" in arrays:
            seen += 1
            assert arrays == ["smem"], (kernel, arrays)
    assert seen
