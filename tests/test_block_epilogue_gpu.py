"""Block-128 products whose CTAs work on many tiles, the last of a row sticking out beyond N: what one tile leaves in the slots of the TMA
stores, the rings and the buffers must not reach the next.  Tolerances are those of test_block_scale_gpu.py."""

import pytest
import torch

from test_block_scale_gpu import BF16, FP16, FP32, _assert_product, _ceil, _dequant, _operands, _runs, _values

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


# width of the tile, rows, columns, K, SMs: every width with several tiles a CTA and the columns of the last that it can have
MANY = [(64, 1500, 8, 128, 3), (64, 1500, 40, 256, 4), (128, 1500, 72, 16, 3), (128, 2600, 104, 256, 4), (192, 2600, 584, 16, 4),
        (192, 2600, 616, 128, 4), (192, 1500, 264, 256, 3), (192, 1500, 296, 128, 4), (192, 1500, 136, 16, 4), (192, 1500, 168, 256, 5),
        (256, 1500, 584, 128, 3), (256, 2600, 616, 16, 3), (256, 1500, 392, 256, 3), (256, 1500, 424, 16, 4), (256, 1500, 200, 128, 4),
        (256, 1500, 232, 256, 5)]


@pytest.mark.parametrize("out", ["bf16", "fp16", "fp32", "odd rows", "behind others"])
@pytest.mark.parametrize("width,m,n,k,sms", MANY)
def test_many_tiles_of_every_width(hq, width, m, n, k, sms, out):
    assert f"128x{width}/128 split=1" in hq.describe_block_tile(m, n, k, sm_count=sms)
    (a, sa), (b, sb) = _operands(hq, m, n, k, m + n + k)
    dtype = {"fp16": FP16, "fp32": FP32}.get(out, BF16)
    ld, skip = {"odd rows": (n + 3, 1), "behind others": (_ceil(n, 8) * 8 + 16, 8)}.get(out, (n, 0))
    ref, first = (_dequant(a, sa), _dequant(b, sb, (128, 128))), None
    for _ in range(3):
        buf = torch.full((m, ld), 7.0, dtype=dtype, device="cuda")
        y = buf[:, skip : skip + n]
        hq.block_gemm(a, b, sa, sb, y, sm_count=sms)
        if first is None:
            first = buf
            _assert_product(y, *ref, _ceil(k, 128))
            assert (buf[:, :skip] == 7).all() and (buf[:, skip + n :] == 7).all()
        assert torch.equal(buf, first)
    assert hq.device_status() == 0


@pytest.mark.parametrize("m,n,k", [(1500, 1040, 16), (700, 1096, 256), (1500, 264, 400), (1500, 136, 1024)])
def test_many_tiles_with_a_scale_per_row_on_both_sides(hq, m, n, k):
    a, sa = hq.block_quant(_values(m, k, m + k))
    b, sb = hq.block_quant(_values(n, k, n + k + 1))
    for dtype in (BF16, FP32):
        first = None
        for _ in range(3):
            out = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
            hq.block_gemm(a, b, sa, sb, out, sm_count=4)
            if first is None:
                first = out
                _assert_product(out, _dequant(a, sa), _dequant(b, sb), _ceil(k, 128))
            assert torch.equal(out, first)
    assert hq.device_status() == 0


EXPERTS = [1300, 0, 257, 2000, 31, 900]


def _assert_rows(y, a, b, k_blocks):
    """_assert_product, with infinities where a result is beyond FP16 (from 65520 on, half a step above its largest value)."""
    if y.dtype == FP16:
        ref, mag = a @ b.t(), a.abs() @ b.abs().t()
        slack = (130 + k_blocks) * 2.0**-23 * mag
        beyond = torch.isinf(y)
        assert (ref.abs()[beyond] >= 65520 - slack[beyond]).all() and (y[beyond] > 0).eq(ref[beyond] > 0).all()
        assert (ref.abs()[~beyond] <= 65520 + slack[~beyond]).all()
        assert beyond.float().mean() < 1e-2
        keep = ~beyond.any(1)
        y, a = y[keep], a[keep]
    _assert_product(y, a, b, k_blocks)


@pytest.mark.parametrize("out", ["bf16", "fp16", "fp32", "odd rows"])
@pytest.mark.parametrize("width,n,k,sms", [(64, 40, 256, 3), (128, 72, 16, 3), (128, 120, 256, 4), (192, 776, 16, 3), (192, 264, 256, 3), (192, 312, 128, 4),
                                           (192, 136, 16, 3), (192, 552, 128, 4), (256, 584, 256, 3), (256, 632, 128, 4), (256, 392, 16, 3),
                                           (256, 440, 128, 3), (256, 712, 16, 5), (256, 488, 256, 4)])
def test_many_tiles_of_experts(hq, width, n, k, sms, out):
    offsets, rows = _runs(EXPERTS)
    assert f"128x{width}/128" in hq.describe_block_tile(rows, n, k, len(EXPERTS), sm_count=sms)
    a, sa = hq.block_quant(_values(rows, k, n))
    b, sb = hq.block_quant(_values(len(EXPERTS) * n, k, n + 1).view(len(EXPERTS), n, k), (128, 128))
    dtype = {"fp16": FP16, "fp32": FP32}.get(out, BF16)
    ld, skip = (n + 3, 1) if out == "odd rows" else (n, 0)
    first, host = None, offsets.tolist()
    for _ in range(3):
        buf = torch.full((rows, ld), 7.0, dtype=dtype, device="cuda")
        y = buf[:, skip : skip + n]
        hq.group_block_gemm(a, b, sa, sb, offsets, y, sm_count=sms)
        if first is None:
            first = buf
            for e, count in enumerate(EXPERTS):
                at = slice(host[e], host[e + 1])
                if count:
                    _assert_rows(y[at], _dequant(a[at], sa[at]), _dequant(b[e], sb[e], (128, 128)), _ceil(k, 128))
            assert (buf[:, :skip] == 7).all() and (buf[:, skip + n :] == 7).all()
        assert torch.equal(buf, first)
    assert hq.device_status() == 0
