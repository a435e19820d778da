"""The weights' gradients of moe_unpermute_backward are sums of h products by 32 or 256 threads with eight sums each.  Each addition loses half a
unit of its result at most, so the gradient is off by (additions of one sum + those that join them) 2^-24 of the sum of the magnitudes.  The values are chosen
so that a longer chain goes over that: one product of 1 at the start of each thread's, and 2^-24 everywhere else, which such a sum drops."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def hq():
    import halops_b200

    return halops_b200


@pytest.mark.parametrize("tokens,threads,h", [(2400, 32, 8192), (3, 256, 65536)], ids=["many pairs", "few pairs"])
@pytest.mark.parametrize("dtype,less,piece", [(BF16, 0, 8), (FP16, 0, 8), (FP32, 0, 4), (BF16, 2, 2), (FP16, 1, 1), (FP32, 1, 1)])
def test_chains_of_the_weights_gradient(hq, tokens, threads, h, dtype, less, piece):
    h -= less  # rows on 16 bytes, on 4, on 2
    order = hq.moe_sort(torch.zeros(tokens, 1, dtype=torch.int32, device="cuda"), 1)
    c = torch.arange(h, device="cuda")
    first = (c < threads * piece) & (c % piece == 0)
    row = torch.where(first, 1.0, 2.0**-12).to(dtype)
    g, z = (row.expand(tokens, h).contiguous() for _ in range(2))
    prod = row.double() ** 2
    _, gw = hq.moe_unpermute_backward(g, z, order, torch.ones(tokens, 1, device="cuda"))
    chain = -(-h // (8 * threads)) + 8  # (and a round of pieces that the row ends in)
    joins = 3 + 5 + threads // 32
    assert ((gw.double() - prod.sum()).abs() <= (chain + joins) * 2.0**-24 * prod.sum()).all(), float((gw.double() / prod.sum() - 1).abs().max() * 2**24)
