"""Calls of the expert-order and SwiGLU entry points that other tests do not make: more slots than a token's rows are read at once, gates whose
bits lie beyond every number, outputs of which one is given."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def hq():
    import halops_b200

    return halops_b200


def _bytes(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("align", [1, 64])
@pytest.mark.parametrize("tokens,topk,experts,h", [(33, 9, 5, 272), (5, 17, 40, 4112), (130, 8, 3, 128), (1, 64, 7, 16)])
def test_many_slots_quantised(hq, tokens, topk, experts, h, align):
    g = torch.Generator().manual_seed(topk)
    ids = torch.randint(-2, experts + 1, (tokens, topk), generator=g).cuda()
    order = hq.moe_sort(ids, experts, align)
    x = (torch.randn(tokens, h, device="cuda") * 50).to(BF16)
    used = int(order.offsets[-1])
    want = hq.block_quant(hq.moe_permute(x, order))
    n = order.pairs.numel()
    q, sf = torch.zeros(n, h, device="cuda").to(torch.float8_e4m3fn), torch.full((n, -(-h // 128)), 3.0, device="cuda")
    hq.moe_permute_block_quant(x, order, output_quant=q, output_sf=sf)
    assert torch.equal(_bytes(q[:used]), _bytes(want[0][:used])) and torch.equal(sf[:used], want[1][:used])
    assert (q[used:].float() == 0).all() and (sf[used:] == 3).all()
    # one of the outputs given
    only_q, new_sf = hq.moe_permute_block_quant(x, order, output_quant=q)
    new_q, only_sf = hq.moe_permute_block_quant(x, order, output_sf=sf)
    assert only_q is q and only_sf is sf
    assert torch.equal(_bytes(new_q[:used]), _bytes(q[:used])) and torch.equal(new_sf[:used], sf[:used])


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_gates_beyond_every_number(hq, dtype):
    x = torch.ones(8, 512, dtype=dtype, device="cuda")
    bits = x.view(torch.int16)
    bits[0, 3] = -1  # a negative NaN: the largest bits of all
    bits[1, 3] = 0x7FFF  # a positive one
    x[2, 3] = float("-inf")
    x[3, 3] = float("inf")
    x[4, 3] = torch.finfo(dtype).min
    x[5, 3], x[5, 259] = -86.0, 3.0
    x[6, 3], x[6, 259] = -87.0, 3.0
    q, sf = hq.swiglu_block_quant(x)
    assert torch.isnan(sf[:3, 0]).all() and torch.isinf(sf[3, 0]) and torch.isfinite(sf[4:]).all() and torch.isfinite(sf[:, 1]).all()
    assert (q[4:7, 3].float() == 0).all()
    others = torch.arange(256, device="cuda") != 3
    assert (q[4:].float()[:, others] == 448).all() and torch.equal(sf[4:], sf[7:].expand(4, 2))
