"""Block-128 products whose CTAs work on many tiles, the last of a row sticking out beyond N: what one tile leaves in the slots of the TMA
stores, the rings and the buffers must not reach the next.  Tolerances are those of test_block_scale_gpu.py."""

import pytest
import torch

from test_block_scale_gpu import BF16, FP16, _assert_product, _ceil, _dequant, _operands, _runs, _values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hq():
    import halops_b200

    return halops_b200


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("m,n,k,sms", [(16384, 264, 128, -1), (16384, 264, 256, -1), (4096, 328, 16, 4), (2000, 264, 256, 4), (4096, 360, 128, 4),
                                       (4096, 648, 128, 4), (4096, 424, 128, 3), (4096, 392, 256, 3), (3000, 456, 16, 3), (4096, 456, 128, 3)])
def test_tiles_after_one_that_sticks_out(hq, m, n, k, sms, dtype):
    (a, sa), (b, sb) = _operands(hq, m, n, k, m + n + k, dtype)
    first = None
    for _ in range(5):
        out = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
        hq.block_gemm(a, b, sa, sb, out, sm_count=sms)
        if first is None:
            first = out
            _assert_product(out, _dequant(a, sa), _dequant(b, sb, (128, 128)), _ceil(k, 128))
        assert torch.equal(out, first)
    assert hq.device_status() == 0


@pytest.mark.parametrize("n,k", [(264, 128), (328, 256), (424, 128), (456, 16)])
def test_experts_tiles_after_one_that_sticks_out(hq, n, k):
    counts = [1300, 0, 257, 2000, 31, 900]
    offsets, rows = _runs(counts)
    a, sa = hq.block_quant(_values(rows, k, n))
    b, sb = hq.block_quant(_values(len(counts) * n, k, n + 1).view(len(counts), n, k), (128, 128))
    first, host = None, offsets.tolist()
    for _ in range(5):
        out = torch.full((rows, n), float("nan"), dtype=BF16, device="cuda")
        hq.group_block_gemm(a, b, sa, sb, offsets, out, sm_count=4)
        first = out if first is None else first
        assert torch.equal(out, first)
    for e in range(len(counts)):
        at = slice(host[e], host[e + 1])
        if counts[e]:
            _assert_product(first[at], _dequant(a[at], sa[at]), _dequant(b[e], sb[e], (128, 128)), _ceil(k, 128))
    assert hq.device_status() == 0
