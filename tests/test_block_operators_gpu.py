"""The block-128 and expert-order entry points at their edges: more than 2^31 elements, both fronts of the Python calls,
launches without programmatic serialisation, streams side by side, values that are not finite."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def hq():
    import halops_b200

    return halops_b200


def _same(a, b):
    return a.dtype == b.dtype and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def _layer(hq, seed, pdl=True, align=1, dtype=BF16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    tokens, topk, experts, h, inner = 75, 3, 9, 384, 208
    x, ids, weights = r(tokens, h).to(dtype), r(tokens, 12).topk(topk, 1).indices - 1, torch.rand(tokens, topk, generator=g, device="cuda")
    w1, w2 = (r(experts, 2 * inner, h) * 0.1).to(dtype), (r(experts, h, inner) * 0.1).to(dtype)
    w1q, w1s = hq.block_quant(w1, (128, 128), use_pdl=pdl)
    w2q, w2s = hq.block_quant(w2, (128, 128), use_pdl=pdl)
    order = hq.moe_sort(ids, experts, align=align, use_pdl=pdl)
    n = order.pairs.numel()
    zeros = lambda c: torch.zeros(n, c, dtype=dtype, device="cuda")  # noqa: E731
    q, sf = hq.moe_permute_block_quant(x, order, use_pdl=pdl)
    mid, down = zeros(2 * inner), zeros(h)
    hq.group_block_gemm(q, w1q, sf, w1s, order.offsets, mid, use_pdl=pdl)
    q2, sf2 = hq.swiglu_block_quant(mid, order.offsets, use_pdl=pdl)
    hq.group_block_gemm(q2, w2q, sf2, w2s, order.offsets, down, use_pdl=pdl)
    y = hq.moe_unpermute(down, order, weights, use_pdl=pdl)
    gz, gw = hq.moe_unpermute_backward(y, down, order, weights, use_pdl=pdl, grad_input=zeros(h))
    xs = hq.moe_permute(x, order, output=zeros(h), use_pdl=pdl)
    gx = hq.moe_permute_backward(gz, order, use_pdl=pdl)
    # and the gradient of a dense layer
    gt, gts = hq.block_quant(y, transpose=True, use_pdl=pdl)
    xt, xts = hq.block_quant(x, transpose=True, use_pdl=pdl)
    gweight = torch.empty(h, h, dtype=FP32, device="cuda")
    hq.block_gemm(gt, xt, gts, xts, gweight, use_pdl=pdl)
    return [*order[:4], mid, down, y, gz, gw, xs, gx, gweight]


@pytest.mark.parametrize("align", [1, 64])
def test_without_programmatic_launches(hq, align):
    for a, b in zip(_layer(hq, 1, True, align), _layer(hq, 1, False, align)):
        assert _same(a, b)


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_both_fronts(hq, monkeypatch, dtype):
    from halops_b200 import _native

    assert _native.load_fast_path() is not _native._NoFastPath
    want = _layer(hq, 2, dtype=dtype)
    monkeypatch.setattr(_native, "fast_path", _native._NoFastPath)
    for a, b in zip(_layer(hq, 2, dtype=dtype), want):
        assert _same(a, b)


def test_two_streams_at_once(hq):
    want = [_layer(hq, s) for s in (3, 4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(_layer(hq, 3 + i))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            assert all(_same(a, b) for a, b in zip(run, want[i]))
    assert hq.device_status() == 0


def test_two_captured_chains_replayed_side_by_side(hq):
    x = torch.randn(40, 256, device="cuda").to(BF16)
    b, sb = hq.block_quant(torch.randn(384, 256, device="cuda").to(BF16), (128, 128))
    want = torch.empty(40, 384, dtype=BF16, device="cuda")
    q, sf = hq.block_quant(x)
    hq.block_gemm(q, b, sf, sb, want)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            q, sf = hq.block_quant(x)
            out = torch.empty(40, 384, dtype=BF16, device="cuda")
            hq.block_gemm(q, b, sf, sb, out)
        graphs.append(graph)
        outs.append(out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


def test_more_than_2_31_elements_quantised(hq):
    m, k = 70016, 32768
    x = torch.empty(m, k, dtype=BF16, device="cuda")
    x[:] = torch.randn(1, k, device="cuda")
    x[-130:] = torch.randn(130, k, device="cuda")
    assert x.numel() > 2**31
    last, want = x[-128:], None
    q, sf = hq.block_quant(x)
    want = hq.block_quant(last.contiguous())
    assert _same(q[-128:], want[0]) and torch.equal(sf[-128:], want[1])
    del q, sf
    q, sf = hq.block_quant(x, (128, 128))
    want = hq.block_quant(last.contiguous(), (128, 128))
    assert _same(q[-128:], want[0]) and torch.equal(sf[-1:], want[1])
    del q, sf
    q, sf = hq.block_quant(x, transpose=True)  # [32768, 70016]
    want = hq.block_quant(last.contiguous(), transpose=True)
    assert _same(q[:, -128:], want[0]) and torch.equal(sf[:, -1:], want[1])


def test_more_than_2_31_elements_of_output(hq):
    m, n = 70016, 32768
    a, sa = hq.block_quant(torch.randn(m, 128, device="cuda").to(BF16))
    b, sb = hq.block_quant(torch.randn(n, 128, device="cuda").to(BF16), (128, 128))
    out = torch.empty(m, n, dtype=BF16, device="cuda")
    hq.block_gemm(a, b, sa, sb, out)
    want = torch.empty(256, n, dtype=BF16, device="cuda")
    hq.block_gemm(a[-256:].contiguous(), b, sa[-256:].contiguous(), sb, want)
    assert torch.equal(out[-256:], want)


def test_more_than_2_31_elements_moved(hq):
    tokens, topk, h = 35000, 8, 8192
    ids = torch.randint(0, 16, (tokens, topk), device="cuda")
    order = hq.moe_sort(ids, 16)
    x = torch.randn(tokens, h, device="cuda").to(BF16)
    rows = hq.moe_permute(x, order)
    assert rows.numel() > 2**31
    for r in (0, tokens * topk // 2, tokens * topk - 1):
        assert torch.equal(rows[r], x[int(order.pairs[r]) // topk])
    # every row is its token's: the sum of topk of them, a power of two, is exact in float32 and in bf16
    assert torch.equal(hq.moe_permute_backward(rows, order), (x.float() * topk).to(BF16))
    weights = torch.ones(tokens, topk, device="cuda")
    gz, _ = hq.moe_unpermute_backward(x, rows, order, weights)
    assert torch.equal(gz, rows)
    del gz
    q, sf = hq.moe_permute_block_quant(x, order)
    for r in (0, tokens * topk - 1):
        want = hq.block_quant(rows[r : r + 1].contiguous())
        assert _same(q[r : r + 1], want[0]) and torch.equal(sf[r : r + 1], want[1])


def test_swiglu_of_values_that_are_not_finite(hq):
    x = torch.ones(5, 512, dtype=BF16, device="cuda")
    x[0, 3] = float("inf")  # gate
    x[1, 256 + 3] = float("nan")  # up
    x[2, 3], x[2, 256 + 3] = -200.0, 5.0  # exp overflows: the product is zero
    x[3, 3] = float("-inf")  # -inf * 0
    q, sf = hq.swiglu_block_quant(x)
    assert torch.isinf(sf[0, 0]) and torch.isnan(sf[1, 0]) and torch.isnan(sf[3, 0])
    assert torch.isfinite(sf[[0, 1, 3], 1]).all() and torch.isfinite(sf[[2, 4]]).all()
    assert q[2, 3].float() == 0 and (q[4].float() == 448).all()


def test_neighbours_that_are_not_finite_do_not_reach_a_run(hq):
    """A tile's copies may bring rows of the next run and weights of the next expert; what they hold stays out of the result."""
    a, sa = hq.block_quant(torch.randn(40, 256, device="cuda").to(BF16))
    w = torch.randn(3, 72, 256, device="cuda").to(BF16)
    b, sb = hq.block_quant(w, (128, 128))
    offsets = torch.tensor([0, 5, 9, 40], dtype=torch.int32, device="cuda")
    want = torch.empty(40, 72, dtype=BF16, device="cuda")
    hq.group_block_gemm(a, b, sa, sb, offsets, want)
    nan_code = 0x7F
    a.view(torch.uint8)[5:9] = nan_code
    sa[5:9] = float("nan")
    b.view(torch.uint8)[1] = nan_code
    sb[1] = float("inf")
    out = torch.empty_like(want)
    hq.group_block_gemm(a, b, sa, sb, offsets, out)
    assert torch.equal(out[:5], want[:5]) and torch.equal(out[9:], want[9:]) and torch.isnan(out[5:9]).all()


def test_outputs_do_not_share_what_they_are_kept_by(hq):
    # codes and scales come from one allocation; writing one leaves the other, and one outlives the other
    x = torch.randn(33, 144, device="cuda").to(BF16)
    q, sf = hq.block_quant(x)
    keep = sf.clone()
    q.view(torch.uint8).fill_(0xFF)
    assert torch.equal(sf, keep)
    del q
    torch.cuda.synchronize()
    junk = [torch.full((1 << 16,), 7, dtype=torch.uint8, device="cuda") for _ in range(50)]
    assert torch.equal(sf, keep) and sf.is_contiguous() and junk[0][0] == 7


def test_a_single_row_may_have_any_stride(hq, monkeypatch):
    from halops_b200 import _native

    _native.load_fast_path()
    column = torch.randn(256, 1, device="cuda").to(BF16)
    row = column.t()
    assert row.shape == (1, 256) and row.stride(0) == 1
    order = hq.moe_sort(torch.tensor([[0, 1]], device="cuda"), 2)
    for front in (_native.fast_path, _native._NoFastPath):
        monkeypatch.setattr(_native, "fast_path", front)
        whole = row.contiguous().clone()
        for block, transpose in (((1, 128), False), ((1, 128), True), ((128, 128), False), ((128, 128), True)):
            got, want = hq.block_quant(row, block, transpose), hq.block_quant(whole, block, transpose)
            assert _same(got[0], want[0]) and torch.equal(got[1], want[1])
        got, want = hq.swiglu_block_quant(row), hq.swiglu_block_quant(whole)
        assert _same(got[0], want[0]) and torch.equal(got[1], want[1])
        got, want = hq.moe_permute_block_quant(row, order), hq.moe_permute_block_quant(whole, order)
        assert _same(got[0], want[0]) and torch.equal(got[1], want[1])
        assert torch.equal(hq.moe_permute(row, order), hq.moe_permute(whole, order))
        assert torch.equal(hq.moe_permute(row.expand(1, 256), order), hq.moe_permute(whole, order))


def test_results_of_the_preceding_kernel_are_waited_for(hq):
    """Programmatic launches back to back, each on what the one before wrote into the same buffers."""
    tokens, topk, h = 512, 2, 256
    ids = torch.empty(tokens, topk, dtype=torch.int64, device="cuda")
    x = torch.empty(tokens, h, dtype=BF16, device="cuda")
    w = torch.randn(4, 128, h, device="cuda").to(BF16)
    wq, ws = hq.block_quant(w, (128, 128))
    out = torch.empty(tokens * topk, 128, dtype=BF16, device="cuda")
    q, sf = torch.empty(tokens * topk, h, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(tokens * topk, h // 128, device="cuda")
    inputs = [(torch.randint(0, 4, (tokens, topk), device="cuda"), torch.randn(tokens, h, device="cuda").to(BF16)) for _ in range(8)]

    def step(pdl):
        order = hq.moe_sort(ids, 4, use_pdl=pdl)
        hq.moe_permute_block_quant(x, order, use_pdl=pdl, output_quant=q, output_sf=sf)
        hq.group_block_gemm(q, wq, sf, ws, order.offsets, out, use_pdl=pdl)
        return hq.moe_unpermute(out, order, use_pdl=pdl)

    want = []
    for i, v in inputs:
        ids.copy_(i)
        x.copy_(v)
        torch.cuda.synchronize()
        want.append(step(False))
        torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for i, v in inputs:
            ids.copy_(i)
            x.copy_(v)
            got.append(step(True))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
