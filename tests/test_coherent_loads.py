"""Kernels that are launched as programmatic dependents may be resident while the
kernel in front still writes what they read.  The non-coherent path (`__ldg`,
`ld.global.nc`, or a `const __restrict__` parameter, which lets the compiler take
it) is defined only for memory that nothing writes during the kernel's whole life."""
import os
import re

import pytest

from conftest import PKG


@pytest.mark.parametrize("name", ["kv_quant.cu", "logprobs.cu"])
def test_no_non_coherent_loads(name):
    with open(os.path.join(PKG, "csrc", name)) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert "pdl_wait_prior_grids" in code
    assert re.findall(r"__ldg\s*\(|global\.nc|__restrict__", code) == []


def kernels(name):
    """(signature, body) of every kernel of a source that waits for the grids in front."""
    with open(os.path.join(PKG, "csrc", name)) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    for m in re.finditer(r"__global__", code):
        start = code.index("{", m.start())
        if ";" in code[m.start():start]:
            continue  # a declaration
        depth, end = 1, start + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(code[end], 0)
            end += 1
        if "pdl_wait_prior_grids" in code[start:end]:
            yield code[m.start():start], code[start:end]


def test_dependent_kernels_read_by_plain_loads():
    """Only weights and tables, which nothing writes between two calls, may be read
    through the non-coherent path by a kernel that the one in front may overlap."""
    found = 0
    for name in sorted(os.listdir(os.path.join(PKG, "csrc"))):
        if not name.endswith(".cu"):
            continue
        for signature, body in kernels(name):
            found += 1
            read_only = re.findall(r"const\s+\w+\s*\*\s*__restrict__\s+(\w+)", signature)
            assert set(read_only) <= {"w", "table"}, (name, signature)
            assert not re.search(r"__ldg\s*\(|global\.nc", body), (name, signature)
    assert found >= 15
    with open(os.path.join(PKG, "csrc", "common.cuh")) as f:
        assert not re.search(r"__ldg\s*\(|global\.nc", re.sub(r"//[^\n]*", "", f.read()))
