"""Sizes that the sort refuses: its kernel counts pairs in 32 bits and steps past the last one, so the bound leaves room for that.  The
arithmetic is followed here in whole numbers; no such size runs on a device."""

import ctypes

import pytest
import torch

import halops_b200 as hq
from halops_b200 import _native, build

P = ctypes.cast(256, ctypes.c_void_p)  # a pointer that a refusal must not follow
LIMIT = 2**31 - 8192


@pytest.fixture(scope="module", autouse=True)
def built():
    build.build()


def _sort(tokens, experts=1, align=1, n_rows=None):
    err = ctypes.create_string_buffer(512)
    n_rows = 2**31 - 1 if n_rows is None else n_rows
    rc = _native.lib().hq_moe_sort(P, 4, tokens, 1, experts, align, n_rows, 0, P, P, P, P, 1 << 20, None, err, 512)
    return rc, err.value.decode()


@pytest.mark.parametrize("pairs", [LIMIT + 1, 2**31 - 4096, 2**31 - 512, 2**31 - 17])
def test_pairs_beyond_the_bound_are_refused(pairs):
    rc, msg = _sort(pairs)
    assert rc == 1 and f"at most 2^31 - 8192 pairs, got {pairs}" in msg
    with pytest.raises(RuntimeError, match=f"at most 2.31 - 8192 pairs, got {pairs}"):
        hq.moe_sort(torch.empty(pairs, 1, dtype=torch.int32, device="meta"), 1)


def test_the_bound_itself_passes_the_check_of_sizes():
    rc, msg = _sort(LIMIT)  # (there is no such device)
    assert rc != 0 and "pairs" not in msg and "rows" not in msg


@pytest.mark.parametrize("ctas", [1, 8, 16])
def test_no_index_of_the_sort_passes_31_bits_at_the_bound(ctas):
    top, warps, held, n = 2**31 - 1, 32, 8, LIMIT
    assert n + 32 * ctas - 1 <= top
    used = min(warps, max(1, (n + 32 * ctas - 1) // (32 * ctas)))
    assert n + ctas * used - 1 <= top
    # a warp's last step past the end of its stretch, and the lanes of a step
    assert n + 32 + 31 <= top and n + held * 32 + 31 <= top
    assert n + 4096 - 1 <= top  # a run's pairs and what pads them
