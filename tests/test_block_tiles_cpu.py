"""The choice of the block-128 products' tile, without a device: every width is some shape's, and refused shapes say so."""

import pytest

import halops_b200 as hq
from halops_b200 import build


@pytest.fixture(scope="module", autouse=True)
def built():
    build.build()


def test_every_width_is_chosen():
    pick = lambda *a, **kw: hq.describe_block_tile(*a, sm_count=148, **kw)  # noqa: E731
    assert "kind=block128 m=8192 n=8192 k=8192 sm=148 -> 128x256/128 split=1" in pick(8192, 8192, 8192)
    assert "128x192/128" in pick(16384, 264, 128)
    assert "128x128/128" in pick(18944, 128, 512)
    assert "128x64/128 split=1" in pick(1, 7168, 2048) and "128x128/128 split=8" in pick(1, 1024, 4096)
    assert "mode=experts kind=block128" in pick(4096, 4096, 2048, num_experts=16)
    for shape in ((8192, 8192, 8192), (7168, 2048, 4096), (200, 64, 128)):
        line = pick(*shape, row_scales=True)
        assert "kind=block128-rows" in line and "split=1" in line and ("128x128/" in line or "128x64/" in line)


@pytest.mark.parametrize("args", [(0, 128, 128), (8, 0, 128), (8, 128, 0), (8, 128, 24), (8, 128, 128, -1), (8, 128, 128, 1025),
                                  (8, 128, 128, 4, True), (1 << 31, 128, 128)])
def test_shapes_without_a_tile(args):
    with pytest.raises(RuntimeError, match="No block-128 tile for M="):
        hq.describe_block_tile(*args, sm_count=148)
