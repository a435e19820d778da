"""FP8 with a float32 scale per block of 128: quantisers against the definition in 64 bits (codes and scales equal), products
against the dequantised operands in 64 bits.

Tolerance of a product: its sums are float32 in steps that lose at most one unit of the last place each (2^-23; 128
within a block, one scaling and one addition per block), relative to the sum of the magnitudes, and the result is rounded once, by at
most half a step of its type."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def hq():
    import halops_b200

    return halops_b200


def _ceil(a, b):
    return -(-a // b)


def _e4m3(v):
    """Nearest e4m3 value of a float64 tensor with |v| <= 448, ties to even."""
    exponent = torch.frexp(v)[1].double() - 1
    step = torch.exp2(exponent.clamp_min(-6.0) - 3)
    return torch.round(v / step) * step


def _pad(x, rows, cols):
    return torch.nn.functional.pad(x, (0, cols - x.size(1), 0, rows - x.size(0)))


def _quant_ref(x, block):
    """(codes as float64, scales as float32) of a matrix."""
    m, k = x.shape
    br, bc = block
    v = _pad(x.double(), _ceil(m, br) * br, _ceil(k, bc) * bc)
    t = v.view(v.size(0) // br, br, v.size(1) // bc, bc)
    amax = t.abs().amax((1, 3)).clamp_min(float(torch.tensor(1e-10, dtype=FP32)))
    q = _e4m3(t * 448 / amax[:, None, :, None]).view_as(v)[:m, :k]
    return q, (amax / 448).float()  # (torch divides a float32 tensor by a number with its reciprocal, so in 64 bits)


def _expand(sf, rows, cols, block):
    return sf.double().repeat_interleave(block[0], 0)[:rows].repeat_interleave(block[1], 1)[:, :cols]


def _dequant(q, sf, block=(1, 128)):
    return q.float().double() * _expand(sf, *q.shape, block)


def _values(m, k, seed, dtype=BF16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, generator=g, device="cuda")
    return (x * torch.exp(torch.randn(m, 1, generator=g, device="cuda"))).to(dtype)


def _assert_product(out, a, b, k_blocks):
    """out against a @ b^T for float64 operands."""
    ref, mag = a @ b.t(), a.abs() @ b.abs().t()
    tol = torch.finfo(out.dtype).eps / 2 * ref.abs() + (130 + k_blocks) * 2.0**-23 * mag
    if out.dtype == FP16:
        tol += 2.0**-25  # half a step of its subnormals
    err = (out.double() - ref).abs()
    assert torch.isfinite(out).all()
    bad = err > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, first at {bad.nonzero()[0].tolist()}, worst {float((err / tol).max()):.2f} of the tolerance"


def _operands(hq, m, n, k, seed, dtype=BF16):
    x, w = _values(m, k, seed, dtype), _values(n, k, seed + 1, dtype) * 0.05
    return hq.block_quant(x), hq.block_quant(w, (128, 128))


# ---------------------------------------------------------------------------- quantisers


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("m,k", [(1, 16), (1, 128), (3, 144), (5, 7168), (130, 272), (257, 1024), (1025, 1040), (4097, 512)])
@pytest.mark.parametrize("block,transpose", [((1, 128), False), ((1, 128), True), ((128, 128), False), ((128, 128), True)],
                         ids=["rows", "rows-t", "tiles", "tiles-t"])
def test_block_quant_is_the_definition(hq, m, k, dtype, block, transpose):
    x = _values(m, k, 7 * m + k, dtype)
    q, sf = hq.block_quant(x, block, transpose)
    want_q, want_sf = _quant_ref(x.t() if transpose else x, block)
    assert q.dtype == torch.float8_e4m3fn and sf.dtype == FP32
    if transpose:
        assert q.shape == (k, _ceil(m, 16) * 16)
        assert (q[:, m:].float() == 0).all()
        q = q[:, :m]
    assert torch.equal(sf, want_sf)
    assert torch.equal(q.float().double(), want_q)


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_values_midway_between_codes(hq, dtype):
    # every maximum of 8 bits against values that fall on midpoints of the codes: ties to even, whatever the maximum
    amax = torch.arange(128, 256, device="cuda", dtype=torch.float64) / 256
    mids = []
    for e in range(-9, 9):
        for f in range(8):
            mids.append((1 + (f + 0.5) / 8) * 2.0**e if e >= -6 else (f + 0.5) * 2.0**-9)
    mids = torch.tensor([m for m in mids if m < 448][:127], dtype=torch.float64, device="cuda")
    x = torch.zeros(128, 128, dtype=torch.float64, device="cuda")
    x[:, 0] = amax
    x[:, 1 : 1 + mids.numel()] = mids * amax[:, None] / 448
    x = x.to(dtype)
    exact = x.double() * 448 / x.double()[:, :1]
    ties = (exact[:, 1:] - _e4m3(exact[:, 1:])).abs() / exact[:, 1:].clamp_min(1e-30)
    assert (ties > 0.01).sum() > 100  # the case is there
    q, sf = hq.block_quant(x)
    want_q, want_sf = _quant_ref(x, (1, 128))
    assert torch.equal(sf, want_sf) and torch.equal(q.float().double(), want_q)


def test_every_16_bit_value_and_its_neighbours(hq):
    for dtype in (BF16, FP16):
        bits = torch.arange(0, 0x7F80 if dtype == BF16 else 0x7C00, device="cuda", dtype=torch.int32).to(torch.int16)
        x = bits.view(dtype)
        x = x[: x.numel() // 128 * 128].view(-1, 128)
        q, sf = hq.block_quant(x)
        want_q, want_sf = _quant_ref(x, (1, 128))
        assert torch.equal(sf, want_sf) and torch.equal(q.float().double(), want_q)


def test_zeros_nans_and_infinities(hq):
    x = torch.ones(4, 256, dtype=BF16, device="cuda")
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 200] = float("-inf")
    for q, sf in (hq.block_quant(x), hq.block_quant(x, (1, 128))):
        assert (q[0].float() == 0).all() and torch.equal(sf[0], (torch.full((2,), 1e-10, device="cuda").double() / 448).float())
        assert torch.isnan(sf[1, 0]) and torch.isnan(q[1, :128].float()).all() and sf[1, 1] == 1 / torch.tensor(448.0)
        assert torch.isinf(sf[2, 1]) and torch.isnan(q[2, 200].float()) and (q[2, 128:200].float() == 0).all()
        assert (q[3].float() == 448).all()
    for transpose in (False, True):
        q, sf = hq.block_quant(x, (128, 128), transpose)
        assert torch.isnan(sf[0, 0]) and torch.isinf(sf.flatten()[1])
    q, sf = hq.block_quant(x, transpose=True)
    assert torch.isnan(sf[5, 0]) and torch.isinf(sf[200, 0]) and sf[6, 0] == 1 / torch.tensor(448.0)


def test_weights_of_several_experts_and_strided_rows(hq):
    x = torch.randn(3, 200, 320, device="cuda").to(BF16)
    for transpose in (False, True):
        q, sf = hq.block_quant(x, (128, 128), transpose)
        for e in range(3):
            one_q, one_sf = hq.block_quant(x[e], (128, 128), transpose)
            assert torch.equal(q[e].view(torch.uint8), one_q.view(torch.uint8)) and torch.equal(sf[e], one_sf)
    wide = torch.randn(64, 1024, device="cuda").to(FP16)
    part = wide[:, 256:640]
    for block, transpose in (((1, 128), False), ((1, 128), True), ((128, 128), False), ((128, 128), True)):
        got, want = hq.block_quant(part, block, transpose), hq.block_quant(part.contiguous(), block, transpose)
        assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])


def test_given_outputs_and_empty_inputs(hq):
    x = _values(9, 256, 3)
    q, sf = torch.empty(9, 256, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(9, 2, device="cuda")
    got = hq.block_quant(x, output_quant=q, output_sf=sf)
    assert got[0] is q and got[1] is sf
    want = hq.block_quant(x)
    assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(sf, want[1])
    empty = hq.block_quant(x[:0])
    assert empty[0].shape == (0, 256) and empty[1].shape == (0, 2)
    empty = hq.swiglu_block_quant(x[:0])
    assert empty[0].shape == (0, 128) and empty[1].shape == (0, 1)


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("m,k", [(1, 16), (3, 128), (17, 144), (130, 2048), (257, 528)])
def test_swiglu_block_quant(hq, m, k, dtype):
    # h is off by 2 |gate| 2^-24 (exp's argument) + 2^-21 (exp, the sum, the quotient, the product) at most: below 1e-5 for |gate| <= 64
    x = (_values(m, 2 * k, m + k, dtype).float().clamp(-60, 60)).to(dtype)
    q, sf = hq.swiglu_block_quant(x)
    gate, up = x.double().chunk(2, 1)
    h = gate * torch.sigmoid(gate) * up
    v = _pad(h, m, _ceil(k, 128) * 128).view(m, -1, 128)
    want_sf = v.abs().amax(2).clamp_min(1e-10) / 448
    assert ((sf.double() - want_sf).abs() <= 1e-5 * want_sf).all()
    got, step = _dequant(q, sf), _expand(sf, m, k, (1, 128))
    assert ((got - h).abs() <= (2.0**-4 + 2e-5) * h.abs() + step * 2.0**-10 * 1.001).all()


def test_swiglu_leaves_rows_behind_the_runs(hq):
    x = _values(40, 512, 11)
    offsets = torch.tensor([0, 7, 7, 23], dtype=torch.int32, device="cuda")
    q = torch.full((40, 256), 1.5, device="cuda").to(torch.float8_e4m3fn)
    sf = torch.full((40, 2), 3.0, device="cuda")
    hq.swiglu_block_quant(x, offsets, output_quant=q, output_sf=sf)
    want = hq.swiglu_block_quant(x)
    assert torch.equal(q[:23].view(torch.uint8), want[0][:23].view(torch.uint8)) and torch.equal(sf[:23], want[1][:23])
    assert (q[23:].float() == 1.5).all() and (sf[23:] == 3.0).all()


# ---------------------------------------------------------------------------- dense products


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 7168, 2048), (2, 129, 144), (7, 64, 128), (16, 2048, 4096), (33, 24576, 1536), (64, 512, 8192),
                                   (65, 1000, 1040), (128, 256, 512), (129, 385, 272), (200, 7168, 2048), (300, 130, 4112), (1000, 4104, 1040),
                                   (2048, 2048, 512), (4096, 1024, 256), (1, 1024, 16384), (128, 128, 7168)])
def test_block_gemm(hq, m, n, k):
    (a, sa), (b, sb) = _operands(hq, m, n, k, m + n + k)
    out = torch.full((m, n), float("nan"), dtype=BF16, device="cuda")
    hq.block_gemm(a, b, sa, sb, out)
    assert hq.device_status() == 0
    _assert_product(out, _dequant(a, sa), _dequant(b, sb, (128, 128)), _ceil(k, 128))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m,n,k", [(1, 24, 256), (130, 264, 400), (96, 1000, 2048), (513, 777, 640)])
def test_block_gemm_output_types_and_strides(hq, m, n, k, dtype):
    (a, sa), (b, sb) = _operands(hq, m, n, k, 5 * m + n)
    ref_a, ref_b = _dequant(a, sa), _dequant(b, sb, (128, 128))
    # rows on 32 bytes, on 16, on single values
    for ld, skip in ((_ceil(n, 16) * 16, 0), (_ceil(n, 8) * 8 + 8, 8), (n + 3, 1)):
        buf = torch.full((m, ld + 16), 7.0, dtype=dtype, device="cuda")
        out = buf[:, skip : skip + n]
        hq.block_gemm(a, b, sa, sb, out)
        _assert_product(out, ref_a, ref_b, _ceil(k, 128))
        assert (buf[:, :skip] == 7).all() and (buf[:, skip + n :] == 7).all()


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (16, 129, 144), (208, 2048, 1024), (130, 300, 4112), (1024, 1040, 208)])
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_block_gemm_with_a_scale_per_row_on_both_sides(hq, m, n, k, dtype):
    a, sa = hq.block_quant(_values(m, k, m + k))
    b, sb = hq.block_quant(_values(n, k, n + k + 1))
    out = torch.full((m, n), float("nan"), dtype=dtype, device="cuda")
    hq.block_gemm(a, b, sa, sb, out)
    assert hq.device_status() == 0
    _assert_product(out, _dequant(a, sa), _dequant(b, sb), _ceil(k, 128))


@pytest.mark.parametrize("m,n,k", [(200, 2048, 1024), (7, 256, 384), (1029, 528, 272)])
def test_backward_of_a_layer(hq, m, n, k):
    """Both gradients against the formulas in 64 bits on the quantised operands, and against differences of the layer's loss."""
    x, w, g = _values(m, k, 1), _values(n, k, 2) * 0.05, _values(m, n, 3) * 0.01
    gq, gs = hq.block_quant(g)
    wt, wts = hq.block_quant(w, (128, 128), transpose=True)
    if n % 16 == 0 and wt.size(1) != n:
        raise AssertionError("transposed weight is padded")
    gx = torch.empty(m, k, dtype=BF16, device="cuda")
    hq.block_gemm(gq, wt, gs, wts, gx)
    wq, ws = hq.block_quant(w, (128, 128))
    wd = _dequant(wq, ws, (128, 128))
    _assert_product(gx, _dequant(gq, gs), wd.t().contiguous(), _ceil(n, 128))
    gt, gts = hq.block_quant(g, transpose=True)
    xt, xts = hq.block_quant(x, transpose=True)
    gw = torch.empty(n, k, dtype=FP32, device="cuda")
    hq.block_gemm(gt, xt, gts, xts, gw)
    assert hq.device_status() == 0
    gd, xd = _dequant(gt, gts)[:, :m], _dequant(xt, xts)[:, :m]
    _assert_product(gw, gd, xd, _ceil(m, 128))
    # loss = <g, x w^T> is bilinear, so its differences along any direction are exact: with the quantised operands for g and x, w
    d = torch.randn(n, k, device="cuda", dtype=torch.float64)
    eps = 2.0**-10
    loss = lambda weight: (gd.t() * (xd.t() @ weight.t())).sum()  # noqa: E731
    difference = (loss(wd + eps * d) - loss(wd - eps * d)) / (2 * eps)
    along = (gw.double() * d).sum()
    scale = (gd.abs() @ xd.abs().t() * d.abs()).sum()
    assert abs(difference - along) <= (131 + _ceil(m, 128)) * 2.0**-23 * scale


def test_non_finite_blocks_reach_their_outputs_alone(hq):
    x, w = _values(70, 512, 1), _values(200, 512, 2)
    x[3, 300] = float("inf")
    a, sa = hq.block_quant(x)
    b, sb = hq.block_quant(w, (128, 128))
    out = torch.empty(70, 200, dtype=BF16, device="cuda")
    hq.block_gemm(a, b, sa, sb, out)
    assert torch.isnan(out[3]).all()
    keep = torch.arange(70, device="cuda") != 3
    _assert_product(out[keep], _dequant(a, sa)[keep], _dequant(b, sb, (128, 128)), 4)


def test_same_bits_every_time_and_on_fewer_sms(hq):
    (a, sa), (b, sb) = _operands(hq, 300, 1000, 4096, 9)
    first = torch.empty(300, 1000, dtype=BF16, device="cuda")
    hq.block_gemm(a, b, sa, sb, first)
    for sms in (-1, -1, 7, 1000):
        out = torch.empty_like(first)
        hq.block_gemm(a, b, sa, sb, out, sm_count=sms)
        if sms == -1:
            assert torch.equal(out, first)
        _assert_product(out, _dequant(a, sa), _dequant(b, sb, (128, 128)), 32)


# ---------------------------------------------------------------------------- experts' products


def _runs(counts, total=None):
    offsets = torch.zeros(len(counts) + 1, dtype=torch.int32)
    offsets[1:] = torch.tensor(counts, dtype=torch.int32).cumsum(0)
    return offsets.cuda(), int(offsets[-1]) if total is None else total


def _group_case(hq, counts, n, k, total=None, dtype=BF16):
    offsets, rows = _runs(counts, total)
    a, sa = hq.block_quant(_values(max(rows, 1), k, sum(counts) + n)[:rows])
    w = _values(len(counts) * n, k, n + k).view(len(counts), n, k)
    b, sb = hq.block_quant(w, (128, 128))
    out = torch.full((rows, n), 3.0, dtype=dtype, device="cuda")
    hq.group_block_gemm(a, b, sa, sb, offsets, out)
    assert hq.device_status() == 0
    host = offsets.tolist()
    for e in range(len(counts)):
        at = slice(host[e], host[e + 1])
        if counts[e]:
            _assert_product(out[at], _dequant(a[at], sa[at]), _dequant(b[e], sb[e], (128, 128)), _ceil(k, 128))
    assert (out[: host[0]] == 3).all() and (out[host[-1] :] == 3).all()


@pytest.mark.parametrize("counts", [[1], [0, 5, 0], [3, 1, 0, 130, 2], [128, 256, 64], [127, 129, 1, 300], [0, 0, 0, 9], [40] * 20, [1000, 0, 17]],
                         ids=lambda c: "-".join(map(str, c[:5])))
@pytest.mark.parametrize("n,k", [(24, 144), (256, 512), (1000, 1040)])
def test_group_block_gemm(hq, counts, n, k):
    _group_case(hq, counts, n, k)


def test_group_block_gemm_with_many_experts_and_rows_behind(hq):
    g = torch.Generator().manual_seed(1)
    _group_case(hq, torch.randint(0, 4, (1024,), generator=g).tolist(), 72, 256)
    _group_case(hq, torch.randint(0, 300, (33,), generator=g).tolist(), 200, 272, total=6000, dtype=FP16)
    _group_case(hq, [0, 0], 64, 128, total=10)
    _group_case(hq, [2500, 1500, 0, 3000], 640, 384, dtype=FP32)


def test_group_runs_that_do_not_start_at_the_first_row(hq):
    a, sa = hq.block_quant(_values(50, 256, 1))
    b, sb = hq.block_quant(_values(2 * 128, 256, 2).view(2, 128, 256), (128, 128))
    out = torch.full((50, 128), 3.0, dtype=BF16, device="cuda")
    hq.group_block_gemm(a, b, sa, sb, torch.tensor([11, 20, 45], dtype=torch.int32, device="cuda"), out)
    for e, at in enumerate((slice(11, 20), slice(20, 45))):
        _assert_product(out[at], _dequant(a[at], sa[at]), _dequant(b[e], sb[e], (128, 128)), 2)
    assert (out[:11] == 3).all() and (out[45:] == 3).all()


def test_group_offsets_out_of_range_are_clamped(hq):
    a, sa = hq.block_quant(_values(50, 256, 1))
    b, sb = hq.block_quant(_values(3 * 128, 256, 2).view(3, 128, 256), (128, 128))
    want = torch.full((50, 128), 3.0, dtype=BF16, device="cuda")
    hq.group_block_gemm(a, b, sa, sb, torch.tensor([0, 20, 20, 50], dtype=torch.int32, device="cuda"), want)
    out = torch.full((60, 128), 3.0, dtype=BF16, device="cuda")
    hq.group_block_gemm(a, b, sa, sb, torch.tensor([-7, 20, 4, 900], dtype=torch.int32, device="cuda"), out[:50])
    assert torch.equal(out[:50], want) and (out[50:] == 3).all()


# ---------------------------------------------------------------------------- streams, graphs, devices


def test_chain_on_another_stream_and_in_a_graph(hq):
    x, w = _values(24, 1024, 1), _values(512, 1024, 2)
    b, sb = hq.block_quant(w, (128, 128))

    def chain():
        a, sa = hq.block_quant(x)
        out = torch.empty(24, 512, dtype=BF16, device="cuda")
        hq.block_gemm(a, b, sa, sb, out)
        return out

    want = chain()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        outs = [chain() for _ in range(5)]
    side.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = chain()
    for seed in (5, 6):
        x.copy_(_values(24, 1024, seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, chain())


def test_refusals_on_the_device(hq):
    (a, sa), (b, sb) = _operands(hq, 8, 128, 256, 1)
    out = torch.empty(8, 128, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError, match=r"sfb must be \[1, 2\]"):
        hq.block_gemm(a, b, sa, sb[:, :1].contiguous(), out)
    with pytest.raises(RuntimeError, match="must match weight K"):
        hq.block_gemm(a, b[:, :128].contiguous(), sa, sb, out)
    with pytest.raises(RuntimeError, match="must be contiguous"):
        hq.block_gemm(a, b, sa.t().contiguous().t(), sb, out)
    with pytest.raises(RuntimeError, match="output rows must be contiguous"):
        hq.block_gemm(a, b, sa, sb, torch.empty(128, 8, dtype=BF16, device="cuda").t())
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        hq.block_gemm(a, b, sa, sb.cpu(), out)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        hq.block_quant(torch.empty(4, 264, dtype=BF16, device="cuda")[:, 1:257])
