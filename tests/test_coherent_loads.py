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
