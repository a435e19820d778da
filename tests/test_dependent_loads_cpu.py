"""Kernels that start while the one before them still runs read its results behind griddepcontrol.wait.  A load that promises the
compiler constant data (__ldg, ld.global.nc, a __restrict__ pointer to const) may be moved to before the wait; none of the block-128 and
expert-order kernels has one."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "halops_b200", "csrc")


@pytest.mark.parametrize("name", ["block_gemm.cu", "block_quant.cu", "block_quant.cuh", "moe.cu"])
def test_no_load_promises_constant_data(name):
    with open(os.path.join(CSRC, name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    assert re.search(r"griddepcontrol\.wait|pdl_wait\(\)|grid_wait\(\)", text)
    assert not re.findall(r"__ldg\b|ld\.global(?:\.\w+)*\.nc\b|__restrict__|__builtin_nontemporal_load", text)
