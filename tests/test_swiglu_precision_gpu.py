"""silu(gate) * up of swiglu_block_quant against 64 bits, read from the scales: one value a block that is not zero, so that
its scale is |h| / 448.

Units of 2^-24 that h can be off by, relative to its value, for a negative gate: exp's 2^-22 and its two last roundings 4 + 1 + 1, the
product with the gate 1, the divisor 1/2 (6) + 1, its reciprocal 2, two products 2: 15.  The scale is rounded once more: 16, or 2^-20.  Below -87
two half exponents and three products, 2 x 6 + 3 + 1, which is 2^-20 too."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def hq():
    import halops_b200

    return halops_b200


def _every(dtype, lo, hi):
    """All values of a 16-bit type in [lo, hi] that are not tiny."""
    x = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x[torch.isfinite(x) & (x.float() >= lo) & (x.float() <= hi) & (x.float().abs() >= 2.0**-8)]
    return x.cuda()


def _scales(hq, gate, up):
    x = torch.zeros(gate.numel(), 256, dtype=gate.dtype, device="cuda")
    x[:, 0], x[:, 128] = gate, up
    q, sf = hq.swiglu_block_quant(x)
    assert (q[:, 0].float().abs() == 448).all() and (q[:, 1:].float() == 0).all()
    assert torch.equal(q[:, 0].float() > 0, (gate.float() > 0) == (up.float() > 0))
    return sf[:, 0].double()


@pytest.mark.parametrize("dtype,lo,hi", [(BF16, -85.0, 300.0), (FP16, -9.0, 2000.0)], ids=["bf16", "fp16"])
def test_every_gate(hq, dtype, lo, hi):
    gate = _every(dtype, lo, hi)
    # a power of two that brings the product near one
    silu = gate.double() * torch.sigmoid(gate.double())
    up = torch.exp2(-torch.floor(torch.log2(silu.abs()))).to(dtype)
    assert torch.isfinite(up).all()
    want = (silu * up.double()).abs() / 448
    sf = _scales(hq, gate, up)
    assert ((sf - want).abs() <= 2.0**-20 * want).all(), float(((sf - want) / want).abs().max())


def test_gates_whose_silu_is_no_normal_number(hq):
    gate = _every(BF16, -105.0, -85.0)
    up = torch.full_like(gate, 2.0**126)
    want = (gate.double() * torch.exp(gate.double()) / (1 + torch.exp(gate.double())) * up.double()).abs() / 448
    assert (want * 448 > 1e-10).all()
    sf = _scales(hq, gate, up)
    assert ((sf - want).abs() <= 2.0**-20 * want).all(), float(((sf - want) / want).abs().max())
    # the smallest of all: nothing is left of the product, whatever `up`
    q, sf = hq.swiglu_block_quant(torch.cat([torch.full((1, 128), -3e38), torch.full((1, 128), 3e38)], 1).to(BF16).cuda())
    assert (q.float() == 0).all() and torch.isfinite(sf).all()


def test_a_far_gate_changes_no_other_value(hq):
    x = (torch.randn(64, 512, device="cuda") * 3).to(BF16)
    x[:, 5::16] = 1.0
    x[:, 256 + 5 :: 16] = 0.0
    q, sf = hq.swiglu_block_quant(x)
    y = x.clone()
    y[:, 5:256:16] = -200.0  # one in each thread's sixteen
    q2, sf2 = hq.swiglu_block_quant(y)
    assert torch.equal(sf, sf2)
    keep = torch.arange(256, device="cuda") % 16 != 5
    assert torch.equal(q.view(torch.uint8)[:, keep], q2.view(torch.uint8)[:, keep]) and (q2.float()[:, ~keep] == 0).all()
