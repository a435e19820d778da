"""Tokens in expert order and back: whole numbers and copies are equal to a plain form's, sums to 64 bits within what float32
sums of that length can lose and one rounding of the result."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def hq():
    import halops_b200

    return halops_b200


def _ids(tokens, topk, lo, hi, seed, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(lo, hi, (tokens, topk), generator=g).to(dtype).cuda()


def _sort_ref(ids, experts, align):
    flat = ids.reshape(-1).tolist()
    runs = [[p for p in range(0)] for _ in range(experts)]
    for p, e in enumerate(flat):
        if 0 <= e < experts:
            runs[e].append(p)
    n = len(flat)
    n_rows = (n + min(experts, n) * (align - 1)) // align * align
    rows, pairs, expert_ids, offsets = [-1] * n, [-1] * n_rows, [experts - 1] * n_rows, [0]
    for e, run in enumerate(runs):
        start = offsets[-1]
        offsets.append(start + -(-len(run) // align) * align)
        for j, p in enumerate(run):
            rows[p], pairs[start + j] = start + j, p
        expert_ids[start : offsets[-1]] = [e] * (offsets[-1] - start)
    t = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return t(rows).view(ids.shape), t(pairs), t(offsets), t(expert_ids)


CASES = [  # tokens, topk, experts, ids from, ids to, align
    (1, 1, 1, 0, 1, 1), (1, 8, 256, 0, 256, 1), (5, 2, 7, -2, 9, 1), (16, 8, 256, 0, 256, 64), (33, 4, 3, 0, 3, 128), (100, 3, 8, 8, 20, 16),
    (513, 8, 64, -64, 64, 64), (1024, 4, 1, 0, 1, 1), (1025, 4, 33, 0, 40, 1), (4096, 2, 16, 0, 16, 128), (3000, 6, 1024, 0, 1024, 1),
    (8192, 8, 128, 0, 256, 64), (20000, 8, 257, 0, 300, 1), (64, 2, 1000, 0, 1000, 300),
]


@pytest.mark.parametrize("tokens,topk,experts,lo,hi,align", CASES)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64], ids=["int32", "int64"])
def test_sort(hq, tokens, topk, experts, lo, hi, align, dtype):
    ids = _ids(tokens, topk, lo, hi, tokens + experts, dtype)
    got = hq.moe_sort(ids, experts, align)
    for name, g, w in zip(got._fields, got, _sort_ref(ids, experts, align)):
        assert torch.equal(g.cpu(), w), name
    assert got.align == align


def test_sort_of_large_ids_and_of_one_expert(hq):
    ids = torch.tensor([[2**40, 1], [-(2**40) + 1, 0], [1 + 2**32, 1]], device="cuda")
    for g, w in zip(hq.moe_sort(ids, 2), _sort_ref(ids, 2, 1)):
        assert torch.equal(g.cpu(), w)
    ids = torch.full((9000, 2), 3, dtype=torch.int32, device="cuda")  # one expert takes everything, each token twice
    for g, w in zip(hq.moe_sort(ids, 5, 64), _sort_ref(ids, 5, 64)):
        assert torch.equal(g.cpu(), w)


def test_sort_without_tokens(hq):
    got = hq.moe_sort(torch.empty(0, 4, dtype=torch.int64, device="cuda"), 3, 64)
    assert got.rows.shape == (0, 4) and got.pairs.shape == (0,) and got.offsets.tolist() == [0, 0, 0, 0]
    x = torch.empty(0, 32, dtype=BF16, device="cuda")
    assert hq.moe_permute(x, got).shape == (0, 32) and hq.moe_unpermute(x, got).shape == (0, 32)
    q, sf = hq.moe_permute_block_quant(x, got)
    assert q.shape == (0, 32) and sf.shape == (0, 1)
    gz, gw = hq.moe_unpermute_backward(x, x, got, torch.empty(0, 4, device="cuda"))
    assert gz.shape == (0, 32) and gw.shape == (0, 4)


MOVES = [  # tokens, topk, experts, ids from, ids to, align, h
    (1, 1, 1, 0, 1, 1, 1), (1, 8, 256, 0, 256, 1, 7168), (5, 2, 7, -2, 9, 1, 33), (97, 2, 7, 0, 7, 64, 1000), (64, 9, 4, 0, 4, 128, 4104),
    (300, 4, 16, -8, 24, 16, 520), (1500, 3, 64, 0, 128, 1, 16), (40, 6, 5, 7, 9, 8, 256), (17, 1, 3, 0, 3, 1, 20000),
]


def _gather_ref(x, order, topk):
    pairs = order.pairs.long()
    got = x[(pairs // topk).clamp_min(0)]
    return torch.where((pairs >= 0)[:, None], got, torch.zeros_like(got))


@pytest.mark.parametrize("tokens,topk,experts,lo,hi,align,h", MOVES)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32, torch.uint8], ids=["bf16", "fp16", "fp32", "uint8"])
def test_permute(hq, tokens, topk, experts, lo, hi, align, h, dtype):
    order = hq.moe_sort(_ids(tokens, topk, lo, hi, h), experts, align)
    x = (torch.randn(tokens, h, device="cuda") * 50).to(dtype)
    used = int(order.offsets[-1])
    want = _gather_ref(x, order, topk)
    out = torch.full((order.pairs.numel(), h), 9, device="cuda").to(dtype)
    assert hq.moe_permute(x, order, output=out) is out
    assert torch.equal(out[:used], want[:used]) and (out[used:] == 9).all()
    assert torch.equal(hq.moe_permute(x, order)[:used], want[:used])
    wide = torch.empty(tokens, h + 5, device="cuda").to(dtype)  # rows on any address
    wide[:, 3 : 3 + h] = x
    assert torch.equal(hq.moe_permute(wide[:, 3 : 3 + h], order)[:used], want[:used])


@pytest.mark.parametrize("tokens,topk,experts,lo,hi,align,h", [c[:6] + (h,) for c, h in zip(CASES, (16, 7168, 144, 7168, 2064, 512, 1024, 128, 48,
                                                                                                   256, 32, 1024, 16, 4096))])
def test_permute_block_quant_is_permute_and_block_quant(hq, tokens, topk, experts, lo, hi, align, h):
    order = hq.moe_sort(_ids(tokens, topk, lo, hi, h), experts, align)
    x = (torch.randn(tokens, h, device="cuda") * 50).to(FP16 if tokens % 2 else BF16)
    used, n_rows = int(order.offsets[-1]), order.pairs.numel()
    want_q, want_sf = hq.block_quant(hq.moe_permute(x, order))
    q = torch.full((n_rows, h), 1.5, device="cuda").to(torch.float8_e4m3fn)
    sf = torch.full((n_rows, -(-h // 128)), 3.0, device="cuda")
    got = hq.moe_permute_block_quant(x, order, output_quant=q, output_sf=sf)
    assert got[0] is q and got[1] is sf
    assert torch.equal(q[:used].view(torch.uint8), want_q[:used].view(torch.uint8)) and torch.equal(sf[:used], want_sf[:used])
    assert (q[used:].float() == 1.5).all() and (sf[used:] == 3.0).all()


@pytest.mark.parametrize("tokens,topk,experts,lo,hi,align,h", MOVES)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("weighted", [True, False], ids=["weights", "ones"])
def test_unpermute_and_its_gradients(hq, tokens, topk, experts, lo, hi, align, h, dtype, weighted):
    order = hq.moe_sort(_ids(tokens, topk, lo, hi, h + 1), experts, align)
    n_rows, used = order.pairs.numel(), int(order.offsets[-1])
    z, g = torch.randn(n_rows, h, device="cuda").to(dtype), torch.randn(tokens, h, device="cuda").to(dtype)
    rows = order.rows.long()
    here = rows >= 0
    z[order.pairs < 0] = float("nan")  # what no pair points to is not read
    weights = torch.rand(tokens, topk, device="cuda") if weighted else None
    if weighted:
        weights[~here] = float("nan")
    w = torch.where(here, weights.double(), 0.0) if weighted else here.double()
    picked = torch.where(here[..., None], z.double()[rows.clamp_min(0)], 0.0)
    eps = torch.finfo(dtype).eps
    tiny = 2.0**-25 if dtype == FP16 else 2.0**-140

    y = hq.moe_unpermute(z, order, weights)
    assert y.dtype == dtype
    want, mag = (w[..., None] * picked).sum(1), (w[..., None] * picked).abs().sum(1)
    assert ((y.double() - want).abs() <= eps / 2 * want.abs() + topk * 2.0**-23 * mag + tiny).all()
    if not weighted:
        assert torch.equal(hq.moe_permute_backward(z, order), y)

    gz = torch.full((n_rows, h), 9, dtype=dtype, device="cuda")
    got = hq.moe_unpermute_backward(g, z, order, weights, grad_input=gz)
    assert got[0] is gz
    pairs = order.pairs.long().clamp_min(0)
    scale = torch.where(order.pairs >= 0, (weights if weighted else torch.ones(tokens, topk, device="cuda")).reshape(-1)[pairs], 0.0)
    want_gz = torch.where((order.pairs >= 0)[:, None], scale[:, None] * g.float()[pairs // topk], 0.0).to(dtype)
    assert torch.equal(gz[:used], want_gz[:used]) and (gz[used:] == 9).all()
    if weighted:
        gw, prod = got[1], picked * g.double()[:, None, :]
        # (a thread adds its values one after another, the threads' sums are joined)
        assert ((gw.double() - prod.sum(2)).abs() <= (h + 16) * 2.0**-24 * prod.abs().sum(2) + 2.0**-140).all()
        assert (gw[~here] == 0).all()
    else:
        assert got[1] is None


def test_gradients_against_differences(hq):
    """y and its loss are linear in the rows and in the weights: differences with steps that are powers of two are exact but
    for the float32 rounding of y."""
    tokens, topk, h = 12, 3, 40
    order = hq.moe_sort(_ids(tokens, topk, -1, 6, 5), 5, 4)
    n_rows = order.pairs.numel()
    z, weights, g = torch.randn(n_rows, h, device="cuda"), torch.rand(tokens, topk, device="cuda"), torch.randn(tokens, h, device="cuda")
    gz, gw = hq.moe_unpermute_backward(g, z, order, weights)
    loss = lambda a, b: (hq.moe_unpermute(a, order, b).double() * g.double()).sum()  # noqa: E731
    bound = 2 * topk * 2.0**-23 * float((g.double().abs() * 8).sum())  # |y| below 8 here
    assert float(hq.moe_unpermute(z, order, weights).abs().max()) < 8
    dz = torch.where((order.pairs >= 0)[:, None], torch.randn(n_rows, h, device="cuda"), 0.0)
    used = order.pairs >= 0
    assert abs((loss(z + dz, weights) - loss(z - dz, weights)) / 2 - (gz.double() * dz.double())[used].sum()) <= 4 * bound
    dw = torch.randn(tokens, topk, device="cuda")
    assert abs((loss(z, weights + dw) - loss(z, weights - dw)) / 2 - (gw.double() * dw.double()).sum()) <= 4 * bound
    # permute: <permute(x), g> = <x, permute_backward(g)>
    x, gp = torch.randn(tokens, h, device="cuda"), torch.randn(n_rows, h, device="cuda")
    left = (hq.moe_permute(x, order).double() * gp.double())[used].sum()
    assert abs(left - (x.double() * hq.moe_permute_backward(gp, order).double()).sum()) <= 4 * bound


def test_strided_rows_and_other_streams(hq):
    order = hq.moe_sort(_ids(50, 2, 0, 6, 3), 6, 8)
    n_rows, used = order.pairs.numel(), int(order.offsets[-1])
    z = torch.randn(n_rows, 300, device="cuda").to(BF16)
    w = torch.rand(50, 2, device="cuda")
    for a, b in ((0, 256), (3, 200)):
        part, whole = z[:, a:b], z[:, a:b].contiguous()
        assert torch.equal(hq.moe_unpermute(part, order, w), hq.moe_unpermute(whole, order, w))
        g = torch.randn(50, 400, device="cuda").to(BF16)[:, a:b]
        got, want = hq.moe_unpermute_backward(g, part, order, w), hq.moe_unpermute_backward(g.contiguous(), whole, order, w)
        assert torch.equal(got[0][:used], want[0][:used])
        assert torch.allclose(got[1], want[1], rtol=0, atol=float((b - a + 16) * 2.0**-23 * 40))
    want = hq.moe_unpermute(z, order, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = hq.moe_unpermute(z, hq.moe_sort(_ids(50, 2, 0, 6, 3), 6, 8), w)
    side.synchronize()
    assert torch.equal(again, want)


def _experts(hq, tokens, topk, experts, h, inner, align, routed, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = r(tokens, h).to(BF16)
    top, ids = r(tokens, routed).topk(topk, dim=1)
    w1, w2 = (r(experts, 2 * inner, h) * 0.05).to(BF16), (r(experts, h, inner) * 0.05).to(BF16)
    return x, ids, torch.softmax(top, 1), w1, w2


@pytest.mark.parametrize("tokens,topk,experts,h,inner,align,routed", [(1, 2, 4, 256, 128, 1, 4), (24, 4, 8, 512, 272, 1, 16),
                                                                    (333, 2, 5, 1040, 400, 64, 5), (1000, 8, 32, 256, 512, 128, 32)])
def test_a_layer_of_experts(hq, tokens, topk, experts, h, inner, align, routed):
    """The run as it is used, stage by stage against 64 bits on what the stage before it gave, and once more in a graph."""
    x, ids, weights, w1, w2 = _experts(hq, tokens, topk, experts, h, inner, align, routed)
    w1q, w1s = hq.block_quant(w1, (128, 128))
    w2q, w2s = hq.block_quant(w2, (128, 128))

    def layer():
        order = hq.moe_sort(ids, experts, align)
        n_rows = order.pairs.numel()
        q, sf = hq.moe_permute_block_quant(x, order)
        mid = torch.zeros(n_rows, 2 * inner, dtype=BF16, device="cuda")
        hq.group_block_gemm(q, w1q, sf, w1s, order.offsets, mid)
        hq_, hs = hq.swiglu_block_quant(mid, order.offsets)
        down = torch.zeros(n_rows, h, dtype=BF16, device="cuda")
        hq.group_block_gemm(hq_, w2q, hs, w2s, order.offsets, down)
        return order, q, sf, mid, hq_, hs, down, hq.moe_unpermute(down, order, weights)

    def dequant(q, sf, block=1):
        return q.float().double() * sf.double().repeat_interleave(block, 0)[: q.size(0)].repeat_interleave(128, 1)[:, : q.size(1)]

    def check(out, a, b):
        ref, mag = a @ b.t(), a.abs() @ b.abs().t()
        assert ((out.double() - ref).abs() <= 2.0**-8 * ref.abs() + (130 + a.size(1) // 128 + 1) * 2.0**-23 * mag).all()

    order, q, sf, mid, h_q, h_s, down, y = layer()
    ends = order.offsets.tolist()
    for e in range(experts):
        at = slice(ends[e], ends[e + 1])
        check(mid[at], dequant(q[at], sf[at]), dequant(w1q[e], w1s[e], 128))
        check(down[at], dequant(h_q[at], h_s[at]), dequant(w2q[e], w2s[e], 128))
    gate, up = mid[: ends[-1]].double().chunk(2, 1)
    want = gate * torch.sigmoid(gate) * up
    got = dequant(h_q[: ends[-1]], h_s[: ends[-1]])
    step = h_s[: ends[-1]].double().repeat_interleave(128, 1)[:, :inner]
    assert ((got - want).abs() <= (2.0**-4 + 2e-5) * want.abs() + step * 2.0**-10 * 1.001).all()
    assert hq.device_status() == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = layer()
    x.copy_(x.roll(1, 0))
    ids.copy_(ids.roll(1, 0))
    weights.copy_(weights.roll(1, 0))
    graph.replay()
    torch.cuda.synchronize()
    # the same tokens in another order: the same rows out
    assert torch.equal(captured[-1].roll(-1, 0), y)


def test_the_order_serves_the_contiguous_gemm(hq):
    """moe_sort(align=64) and moe_permute in front of group_wise_quant and group_contiguous_gemm."""
    tokens, topk, experts, h, n = 200, 3, 6, 512, 256
    x, ids, weights, w, _ = _experts(hq, tokens, topk, experts, h, n // 2, 64, experts)
    order = hq.moe_sort(ids, experts, align=64)
    xs = hq.moe_permute(x, order, output=torch.zeros(order.pairs.numel(), h, dtype=BF16, device="cuda"))
    parts = [hq.group_wise_quant(w[e]) for e in range(experts)]
    wq, ws = torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])
    q, sf = hq.group_wise_quant(xs)
    out = torch.empty(order.pairs.numel(), n, dtype=BF16, device="cuda")
    hq.group_contiguous_gemm(q, wq, sf, ws, order.expert_ids, out)
    assert hq.device_status() == 0
    y = hq.moe_unpermute(out, order, weights)
    want = torch.zeros(tokens, n, dtype=torch.float64, device="cuda")
    for s in range(topk):
        want += weights[:, s : s + 1].double() * torch.einsum("th,tnh->tn", x.double(), w.double()[ids[:, s]])
    # MXFP8 codes are off by 2^-4 of a value at most, the products of 512 such pairs by far less of their result
    assert (y.double() - want).norm() <= 0.05 * want.norm()


def test_refusals_on_the_device(hq):
    order = hq.moe_sort(_ids(8, 2, 0, 4, 1), 4)
    x = torch.zeros(8, 32, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError, match="8 tokens, got 7"):
        hq.moe_permute(x[:7], order)
    with pytest.raises(RuntimeError, match="16 rows, got 8"):
        hq.moe_unpermute(x, order)
    with pytest.raises(RuntimeError, match=r"weights must be a contiguous float32 tensor of shape \[8, 2\]"):
        hq.moe_unpermute(torch.zeros(16, 32, dtype=BF16, device="cuda"), order, torch.ones(8, 2, dtype=BF16, device="cuda"))
    with pytest.raises(RuntimeError, match="hidden size must be divisible by 16"):
        hq.moe_permute_block_quant(torch.zeros(8, 40, dtype=BF16, device="cuda"), order)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        hq.moe_permute(x, order._replace(rows=order.rows.cpu()))
    with pytest.raises(RuntimeError, match="grad_output must be"):
        hq.moe_unpermute_backward(x.float(), torch.zeros(16, 32, dtype=BF16, device="cuda"), order)
    with pytest.raises(RuntimeError, match="topk_ids must be contiguous"):
        hq.moe_sort(_ids(2, 8, 0, 4, 1).t(), 4)
