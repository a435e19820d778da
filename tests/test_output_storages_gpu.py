"""Codes and scales that a quantiser returns are tensors of their own: each has a storage of its size, is saved alone, and outlives the
other's storage, on both fronts of the Python calls."""

import io

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hq():
    import halops_b200

    return halops_b200


@pytest.fixture(params=["native", "python"])
def front(request, monkeypatch):
    from halops_b200 import _native

    _native.load_fast_path()
    if request.param == "python":
        monkeypatch.setattr(_native, "fast_path", _native._NoFastPath)


def _calls(hq):
    x = torch.randn(64, 4096, device="cuda").to(torch.bfloat16)
    order = hq.moe_sort(torch.randint(0, 4, (64, 2), device="cuda"), 4)
    return {"block_quant": lambda: hq.block_quant(x), "block_quant of tiles": lambda: hq.block_quant(x, (128, 128), True),
            "swiglu_block_quant": lambda: hq.swiglu_block_quant(x), "moe_permute_block_quant": lambda: hq.moe_permute_block_quant(x, order)}


@pytest.mark.parametrize("name", ["block_quant", "block_quant of tiles", "swiglu_block_quant", "moe_permute_block_quant"])
def test_codes_and_scales_have_a_storage_each(hq, front, name):
    call = _calls(hq)[name]
    q, sf = call()
    keep = sf.clone()
    for t in (q, sf):
        assert t.storage_offset() == 0 and t.untyped_storage().nbytes() == t.numel() * t.element_size()
    file = io.BytesIO()
    torch.save(sf, file)
    assert len(file.getvalue()) < sf.numel() * 4 + 4096
    torch.cuda.synchronize()
    q.untyped_storage().resize_(0)  # a caller that frees the codes
    assert sf.data_ptr() != 0 and torch.equal(sf, keep)


def test_scales_alone_keep_their_own_bytes(hq, front):
    x = torch.randn(4096, 4096, device="cuda").to(torch.bfloat16)
    hq.block_quant(x)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    scales = [hq.block_quant(x)[1] for _ in range(4)]
    assert torch.cuda.memory_allocated() - before <= 4 * (scales[0].numel() * 4 + 4096)
