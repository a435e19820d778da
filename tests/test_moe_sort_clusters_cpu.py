"""A cluster of 16 CTAs is more than every device has to hold (a partition of one, a context with few SMs), so the sort asks for room before
it takes one and has 8 to go back to.  The sort gives the same with either (tests/test_moe_gpu.py); that the launch asks
is read from the source, since no device here is partitioned."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "halops_b200", "csrc")


def test_a_cluster_of_16_is_taken_where_there_is_room():
    with open(os.path.join(CSRC, "moe.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    launch = text[text.index("cudaError_t launch_sort("):]
    launch = launch[: launch.index("\n}")]
    assert re.search(r"int ctas = pairs_n > 16384 \? 16 :", launch)
    opt_in, ask, go_back, start = (launch.index(s) for s in ("cudaFuncAttributeNonPortableClusterSizeAllowed", "cluster16_fits<Id>(opt, dev, bytes, &fits)",
                                                             "if (!fits) ctas = 8;", "return launch(moe_sort_kernel<Id>"))
    assert opt_in < ask < go_back < start
    fits = text[text.index("cudaError_t cluster16_fits("): text.index("cudaError_t launch_sort(")]
    assert "cudaOccupancyMaxActiveClusters(&clusters, moe_sort_kernel<Id>, &cfg)" in fits


def test_the_number_of_sms_is_the_devices():
    with open(os.path.join(CSRC, "moe.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    assert not re.search(r"\b(148|132|144|160)\b", text) and "n >= int64_t(sms) * 16" in text and "sms = hq_sm_count(device)" in text
