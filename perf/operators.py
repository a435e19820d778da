"""Measured operators: FP8 products with a scale for each block of 128, and tokens sorted by expert and back.

Five kinds of pass, each the calls that a layer makes:

  linear      16-bit rows are quantised in blocks of 1 x 128 and multiplied with a weight that is kept in FP8 with a
              scale for each block of 128 x 128
  grad        the backward pass of such a layer: the gradient of its input through the transposed weight, the
              gradient of its weight from the layer's input and the output's gradient, both in FP8
  dispatch    tokens sorted by the experts that a router gave them, gathered and quantised in expert order
  exchange    training of a mixture of experts: tokens to expert order, the experts' rows back with the router's
              weights, and the gradients of both
  experts     the whole block: sort, gather and quantise, gate and up product, SwiGLU, down product, back with weights

The plain forms compute in 32 bits with elementary operations.  Where a value is quantised, x * 448 is exact in 32 bits
for 16-bit x, and the quotient by the block's maximum is rounded correctly, so that values midway between
two codes stay midway.

The expert-ordered buffers have room for any ids that a router can give (``_rows``).  They belong to the program, and what lies behind
the last expert's run stays as it is, here zero.
"""

import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
AMAX_FLOOR = 1e-10
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _linear(name, m, n, k, dtype="bf16"):
    return {"name": name, "kind": "linear", "m": m, "n": n, "k": k, "dtype": dtype}


def _grad(name, m, n, k, dtype="bf16"):
    return {"name": name, "kind": "grad", "m": m, "n": n, "k": k, "dtype": dtype}


def _moe(name, kind, tokens, hidden, topk, experts, routed, align=1, inner=0, dtype="bf16"):
    """``routed`` experts that the router chooses among, of which ``experts`` are here (the others' pairs are dropped)."""
    return {"name": name, "kind": kind, "tokens": tokens, "hidden": hidden, "topk": topk, "experts": experts,
            "routed": routed, "align": align, "inner": inner, "dtype": dtype}


def listed():
    return [
        # one token of a decode step through a projection
        _linear("linear-1x7168x2048", 1, 7168, 2048),
        # a decode batch through a wide projection: the weight's bytes count
        _linear("linear-32x24576x1536", 32, 24576, 1536),
        # a prompt of 1000 tokens in FP16, widths that fill no tile and no block
        _linear("linear-1000x4104x4112", 1000, 4104, 4112, "fp16"),
        # large square problem
        _linear("linear-8192x8192x8192", 8192, 8192, 8192),
        # backward of a small layer on a short ragged batch
        _grad("grad-200x2048x1024", 200, 2048, 1024),
        # backward of a projection on 4096 tokens
        _grad("grad-4096x7168x2048", 4096, 7168, 2048),
        # decode step of a wide mixture of experts: launches count
        _moe("dispatch-16x7168-top8of256", "dispatch", 16, 7168, 8, 256, 256),
        # prefill with half of the experts on this device, runs padded for tiles of 64 rows
        _moe("dispatch-8192x4096-top8of128", "dispatch", 8192, 4096, 8, 64, 128, align=64),
        # a short training batch over few experts, FP16, odd sizes
        _moe("exchange-97x1000-top2of7", "exchange", 97, 1000, 2, 7, 7, dtype="fp16"),
        # a training batch: sorted, back, and both gradients
        _moe("exchange-8192x4096-top4of64", "exchange", 8192, 4096, 4, 64, 64),
        # decode batch through all experts: their weights' bytes count
        _moe("experts-24x4096x1024-top4of32", "experts", 24, 4096, 4, 32, 32, inner=1024),
        # prefill through the experts: their products count
        _moe("experts-4096x4096x2048-top4of16", "experts", 4096, 4096, 4, 16, 16, inner=2048),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of ``step`` in [lo, hi], evenly spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi // step * step, max(-(-lo // step) * step, round(v / step) * step)))


def draw(rng):
    while True:
        kind = rng.choice(["linear", "linear", "grad", "dispatch", "exchange", "experts"])
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        if kind == "linear":
            c = _linear("", _log(rng, 1, 8192), _log(rng, 256, 24576, rng.choice([1, 8, 128])), _log(rng, 512, 8192, 16), dtype)
        elif kind == "grad":
            c = _grad("", _log(rng, 1, 8192), _log(rng, 256, 8192, 16), _log(rng, 256, 8192, 16), dtype)
        else:
            experts = rng.choice([1, 4, 7, 8, 16, 32, 64, 128, 256] if kind != "experts" else [4, 7, 8, 16, 32])
            routed = experts * rng.choice([1, 1, 2, 4])
            c = _moe("", kind, _log(rng, 1, 8192), _log(rng, 512, 8192, 16 if kind != "exchange" else rng.choice([1, 8])),
                     min(routed, rng.choice([1, 2, 4, 6, 8])), experts, routed, align=rng.choice([1, 1, 64, 128]),
                     inner=_log(rng, 512, 4096, 16) if kind == "experts" else 0, dtype=dtype)
        w = work(c)
        # nothing above the large square problem and the largest exchange
        if w["flops"] <= 2 * 8192**3 and w["bytes"] <= 1.2e9:
            return c


def _rows(case):
    """Rows of the expert-ordered buffers: a bound that holds for any ids, a multiple of the alignment."""
    pairs, align = case["tokens"] * case["topk"], case["align"]
    return (pairs + min(case["experts"], pairs) * (align - 1)) // align * align


def work(case):
    if case["kind"] in ("linear", "grad"):
        m, n, k = case["m"], case["n"], case["k"]
        if case["kind"] == "linear":
            return {"bytes": 2 * m * k + n * k * (1 + 4 / BLOCK**2) + 2 * m * n, "flops": 2 * m * n * k}
        return {"bytes": 2 * m * n + 2 * m * k + n * k * (1 + 4 / BLOCK**2) + 2 * m * k + 4 * n * k, "flops": 4 * m * n * k}
    t, h, k, e = case["tokens"], case["hidden"], case["topk"], case["experts"]
    here = t * k * e / case["routed"]  # pairs whose expert is on this device
    if case["kind"] == "dispatch":
        r = _rows(case)
        return {"bytes": 2 * t * h + here * h * (1 + 4 / BLOCK) + 4 * (3 * t * k + 2 * r + e), "flops": here * h}
    if case["kind"] == "exchange":
        # x, the experts' rows, the two gradients in; rows, tokens and the three gradients out
        return {"bytes": 2 * h * (4 * t + 4 * here) + 4 * t * k, "flops": 6 * here * h}
    i = case["inner"]
    active = e * (1 - (1 - k / case["routed"]) ** t)
    return {"bytes": 4 * t * h + active * 3 * i * h + 2 * here * (2 * i + h), "flops": 6 * here * i * h}


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _activation(g, m, k, dtype):
    """Rows of a residual stream: channels and rows of different size, a few channels far above the others."""
    scale = torch.exp(0.5 * _normal(g, 1, k)) * torch.where(torch.rand(1, k, generator=g, device="cuda") < 0.004, 20.0, 1.0)
    return (_normal(g, m, k) * scale * torch.exp(0.3 * _normal(g, m, 1))).to(_DTYPES[dtype])


def _fp8_weight(g, *shape):
    """A weight as it is kept: e4m3 codes [.., n, k] and a float32 scale for each block of 128 x 128."""
    n, k = shape[-2:]
    w = (_normal(g, *shape) * 0.02).to(torch.bfloat16).float()
    pad = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK))
    tiles = pad.unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, BLOCK))
    amax = tiles.abs().amax((-3, -1)).clamp_min(AMAX_FLOOR)
    q = tiles * E4M3_MAX / amax[..., :, None, :, None]
    q = q.flatten(-2).flatten(-3, -2)[..., :n, :k].to(torch.float8_e4m3fn)
    return q.contiguous(), amax / E4M3_MAX


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": dict(case)}
    if case["kind"] in ("linear", "grad"):
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = _activation(g, m, k, case["dtype"])
        s["w"], s["sw"] = _fp8_weight(g, n, k)
        if case["kind"] == "grad":
            # the gradient of the output, and the weight as the backward pass reads it
            s["g"] = (_normal(g, m, n) * torch.exp(0.5 * _normal(g, m, 1)) * 1e-2).to(_DTYPES[case["dtype"]])
            s["wt"], s["swt"] = s.pop("w").t().contiguous(), s.pop("sw").t().contiguous()
        return s
    t, h, k, e = case["tokens"], case["hidden"], case["topk"], case["experts"]
    # some experts are liked more than others
    logits = _normal(g, t, case["routed"]) + 0.7 * _normal(g, 1, case["routed"])
    top, ids = logits.topk(k, dim=1)
    s["ids"] = ids - (case["routed"] - e) // 2  # ids outside of [0, experts) belong to another device
    s["weights"] = torch.softmax(top, dim=1)
    s["x"] = _activation(g, t, h, case["dtype"])
    r, dtype = _rows(case), _DTYPES[case["dtype"]]
    if case["kind"] != "exchange":
        s["q"] = torch.zeros(r, h, device="cuda").to(torch.float8_e4m3fn)
        s["sf"] = torch.zeros(r, -(-h // BLOCK), device="cuda")
    if case["kind"] == "exchange":
        s["xs"], s["gz"] = (torch.zeros(r, h, dtype=dtype, device="cuda") for _ in range(2))
        s["z"] = _normal(g, r, h).to(_DTYPES[case["dtype"]])
        s["gy"] = _normal(g, t, h).to(_DTYPES[case["dtype"]])
        s["gxs"] = _normal(g, r, h).to(_DTYPES[case["dtype"]])
    if case["kind"] == "experts":
        i = case["inner"]
        s["w1"], s["sw1"] = _fp8_weight(g, e, 2 * i, h)
        s["w2"], s["sw2"] = _fp8_weight(g, e, h, i)
        s["mid"], s["down"] = (torch.zeros(r, c, dtype=dtype, device="cuda") for c in (2 * i, h))
    return s


# ---------------------------------------------------------------------------- the framework's operators


def _run_own(s):
    import halops_b200 as hq

    case = s["case"]
    kind, dtype = case["kind"], _DTYPES[case["dtype"]]
    if kind == "linear":
        q, sf = hq.block_quant(s["x"])
        out = torch.empty(case["m"], case["n"], dtype=dtype, device="cuda")
        hq.block_gemm(q, s["w"], sf, s["sw"], out)
        return out
    if kind == "grad":
        q, sf = hq.block_quant(s["g"])
        gx = torch.empty(case["m"], case["k"], dtype=dtype, device="cuda")
        hq.block_gemm(q, s["wt"], sf, s["swt"], gx)
        gt, sgt = hq.block_quant(s["g"], transpose=True)
        xt, sxt = hq.block_quant(s["x"], transpose=True)
        gw = torch.empty(case["n"], case["k"], dtype=torch.float32, device="cuda")
        hq.block_gemm(gt, xt, sgt, sxt, gw)
        return gx, gw
    order = hq.moe_sort(s["ids"], case["experts"], align=case["align"])
    if kind == "dispatch":
        q, sf = hq.moe_permute_block_quant(s["x"], order, output_quant=s["q"], output_sf=s["sf"])
        return order.rows, order.pairs, order.offsets, order.expert_ids, q, sf
    if kind == "exchange":
        xs = hq.moe_permute(s["x"], order, output=s["xs"])
        y = hq.moe_unpermute(s["z"], order, s["weights"])
        gz, gweights = hq.moe_unpermute_backward(s["gy"], s["z"], order, s["weights"], grad_input=s["gz"])
        gx = hq.moe_permute_backward(s["gxs"], order)
        return xs, y, gz, gweights, gx
    q, sf = hq.moe_permute_block_quant(s["x"], order, output_quant=s["q"], output_sf=s["sf"])
    hq.group_block_gemm(q, s["w1"], sf, s["sw1"], order.offsets, s["mid"])
    q, sf = hq.swiglu_block_quant(s["mid"], offsets=order.offsets)
    hq.group_block_gemm(q, s["w2"], sf, s["sw2"], order.offsets, s["down"])
    return s["mid"], s["down"], hq.moe_unpermute(s["down"], order, s["weights"])


# ---------------------------------------------------------------------------- plain forms


def _plain_quant(x):
    """[m, k] -> e4m3 codes and one float32 scale for each 128 values of a row."""
    m, k = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -k % BLOCK)).view(m, -1, BLOCK)
    amax = v.abs().amax(-1).clamp_min(AMAX_FLOOR)
    q = (v * E4M3_MAX / amax[..., None]).view(m, -1)[:, :k].to(torch.float8_e4m3fn)
    return q, amax / E4M3_MAX


def _plain_rows(q, sf):
    """The values that rows quantised in blocks of 1 x 128 stand for."""
    return q.float() * sf.repeat_interleave(BLOCK, 1)[:, : q.size(1)]


def _plain_weight(q, sf):
    """The values that a weight quantised in blocks of 128 x 128 stands for."""
    return q.float() * sf.repeat_interleave(BLOCK, 0)[: q.size(0)].repeat_interleave(BLOCK, 1)[:, : q.size(1)]


def _plain_sort(ids, experts, align, n_rows):
    pairs_n = ids.numel()
    flat = ids.reshape(-1).long()
    here = (flat >= 0) & (flat < experts)
    key = torch.where(here, flat, experts)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device).scatter_add_(0, key, torch.ones_like(key))[:experts]
    padded = (counts + align - 1) // align * align
    zero = torch.zeros(1, dtype=torch.int64, device=ids.device)
    offsets = torch.cat([zero, padded.cumsum(0)])
    starts = torch.cat([zero, counts.cumsum(0)])
    order = key.argsort(stable=True)  # pairs by expert; equal experts in the order of the tokens
    by = key[order]
    place = offsets[by] + torch.arange(pairs_n, device=ids.device) - starts[by]
    place = torch.where(by < experts, place, n_rows)  # dropped pairs: one place behind the rows
    rows = torch.empty_like(flat).scatter_(0, order, torch.where(by < experts, place, -1)).view(ids.shape)
    pairs = torch.full((n_rows + 1,), -1, dtype=torch.int64, device=ids.device).scatter_(0, place, order)[:n_rows]
    at = torch.arange(n_rows, device=ids.device)
    expert_ids = torch.searchsorted(offsets[1:].contiguous(), at, right=True).clamp_max(experts - 1)
    return rows.int(), pairs.int(), offsets.int(), expert_ids.int()


def _plain_gather(x, pairs, topk):
    got = x[(pairs.long() // topk).clamp_min(0)]
    return torch.where((pairs >= 0)[:, None], got, torch.zeros_like(got))


def _plain_scatter_back(z, rows, weights):
    """sum over a token's experts of weight * row, in 32 bits (pairs without a row count as zero)."""
    here = rows >= 0
    got = z.float()[rows.long().clamp_min(0)]  # [tokens, topk, hidden]
    got = torch.where(here[..., None], got, 0.0)
    if weights is not None:
        got = got * torch.where(here, weights, 0.0)[..., None]
    return got.sum(1)


def _plain_grouped(q, sf, w, sw, offsets, dtype):
    out = torch.zeros(q.size(0), w.size(1), dtype=dtype, device=q.device)
    ends = offsets.tolist()
    for e in range(w.size(0)):
        a, b = ends[e], ends[e + 1]
        if b > a:
            out[a:b] = (_plain_rows(q[a:b], sf[a:b]) @ _plain_weight(w[e], sw[e]).t()).to(dtype)
    return out


def _plain_swiglu(mid):
    gate, up = mid.float().chunk(2, dim=1)
    return gate / (1 + torch.exp(-gate)) * up


def _run_plain(s):
    case = s["case"]
    kind, dtype = case["kind"], _DTYPES[case["dtype"]]
    if kind == "linear":
        return (_plain_rows(*_plain_quant(s["x"])) @ _plain_weight(s["w"], s["sw"]).t()).to(dtype)
    if kind == "grad":
        gx = (_plain_rows(*_plain_quant(s["g"])) @ _plain_weight(s["wt"], s["swt"]).t()).to(dtype)
        return gx, _plain_rows(*_plain_quant(s["g"].t())) @ _plain_rows(*_plain_quant(s["x"].t())).t()
    topk = case["topk"]
    rows, pairs, offsets, expert_ids = _plain_sort(s["ids"], case["experts"], case["align"], _rows(case))
    if kind == "dispatch":
        q, sf = _plain_quant(_plain_gather(s["x"], pairs, topk))
        in_runs = torch.arange(sf.size(0), device=sf.device) < offsets[-1]
        return rows, pairs, offsets, expert_ids, q, torch.where(in_runs[:, None], sf, 0.0)
    if kind == "exchange":
        xs = _plain_gather(s["x"], pairs, topk)
        y = _plain_scatter_back(s["z"], rows, s["weights"]).to(dtype)
        # a row's gradient is its token's times the pair's weight; a weight's is the row's product with its token's gradient
        scale = torch.where(pairs >= 0, s["weights"].reshape(-1)[pairs.long().clamp_min(0)], 0.0)
        gz = (_plain_gather(s["gy"], pairs, topk).float() * scale[:, None]).to(dtype)
        got = s["z"].float()[rows.long().clamp_min(0)]
        gweights = torch.where(rows >= 0, (got * s["gy"].float()[:, None, :]).sum(-1), 0.0)
        return xs, y, gz, gweights, _plain_scatter_back(s["gxs"], rows, None).to(dtype)
    mid = _plain_grouped(*_plain_quant(_plain_gather(s["x"], pairs, topk)), s["w1"], s["sw1"], offsets, dtype)
    down = _plain_grouped(*_plain_quant(_plain_swiglu(mid)), s["w2"], s["sw2"], offsets, dtype)
    return mid, down, _plain_scatter_back(down, rows, s["weights"]).to(dtype)


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ---------------------------------------------------------------------------- the definition, in 64 bits


def _e4m3(v):
    """The e4m3 value nearest to v (|v| <= 448), ties to the even code: three bits behind the leading one, steps of
    2^-9 below 2^-6."""
    exponent = torch.frexp(v)[1].to(torch.float64) - 1
    step = torch.exp2(exponent.clamp_min(-6.0) - 3)
    return torch.round(v / step) * step


def _exact_quant(x):
    """Codes (as values) and scales of rows in blocks of 128."""
    m, k = x.shape
    codes, scales = torch.empty(m, k, dtype=torch.float64, device=x.device), []
    for b in range(0, k, BLOCK):
        v = x[:, b : b + BLOCK].double()
        amax = torch.maximum(v.abs().max(1).values, torch.tensor(AMAX_FLOOR, dtype=torch.float64, device=x.device))
        codes[:, b : b + BLOCK] = _e4m3(v * E4M3_MAX / amax[:, None])
        scales.append(amax / E4M3_MAX)
    return codes, torch.stack(scales, 1)


def _exact_rows(x):
    codes, scales = _exact_quant(x)
    for b in range(scales.size(1)):
        codes[:, b * BLOCK : (b + 1) * BLOCK] *= scales[:, b : b + 1]
    return codes


def _exact_weight(q, sf):
    w = q.float().double()
    for i in range(sf.size(0)):
        row = sf[i].double().repeat_interleave(BLOCK)[: q.size(1)]
        w[i * BLOCK : (i + 1) * BLOCK] *= row
    return w


def _exact_sort(case, ids):
    """Lists of the pairs of each expert in token order, and the row where each expert's run begins."""
    flat = ids.reshape(-1).cpu().tolist()
    mine = [[] for _ in range(case["experts"])]
    for p, e in enumerate(flat):
        if 0 <= e < case["experts"]:
            mine[e].append(p)
    offsets = [0]
    for run_ in mine:
        offsets.append(offsets[-1] + -(-len(run_) // case["align"]) * case["align"])
    return mine, offsets


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "linear":
        return _exact_rows(s["x"]) @ _exact_weight(s["w"], s["sw"]).t()
    if kind == "grad":
        gx = _exact_rows(s["g"]) @ _exact_weight(s["wt"], s["swt"]).t()
        return gx, _exact_rows(s["g"].t()) @ _exact_rows(s["x"].t()).t()
    topk, n_rows = case["topk"], _rows(case)
    mine, offsets = _exact_sort(case, s["ids"])
    dev = s["x"].device
    rows, pairs, expert_ids = [-1] * (case["tokens"] * topk), [-1] * n_rows, [case["experts"] - 1] * n_rows
    for e, run_ in enumerate(mine):
        expert_ids[offsets[e] : offsets[e + 1]] = [e] * (offsets[e + 1] - offsets[e])
        for j, p in enumerate(run_):
            rows[p], pairs[offsets[e] + j] = offsets[e] + j, p
    as_int = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    pairs_t, rows_t = as_int(pairs).long(), as_int(rows).long()
    valid = pairs_t >= 0
    gathered = torch.zeros(n_rows, case["hidden"], dtype=torch.float64, device=dev)
    gathered[valid] = s["x"].double()[pairs_t[valid] // topk]
    if kind == "dispatch":
        codes, scales = _exact_quant(gathered)
        scales[offsets[-1]:] = 0
        return as_int(rows).view(-1, topk), as_int(pairs), as_int(offsets), as_int(expert_ids), codes, scales
    weights = s["weights"].double().reshape(-1)
    tokens = torch.arange(case["tokens"] * topk, device=dev) // topk
    used = rows_t >= 0
    if kind == "exchange":
        y = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device=dev)
        y.index_add_(0, tokens[used], weights[used, None] * s["z"][rows_t[used]].double())
        gx = torch.zeros_like(y)
        gx.index_add_(0, tokens[used], s["gxs"][rows_t[used]].double())
        gz = torch.zeros_like(gathered)
        gz[rows_t[used]] = weights[used, None] * s["gy"][tokens[used]].double()
        gweights = torch.zeros_like(weights)
        gweights[used] = (s["z"][rows_t[used]].double() * s["gy"][tokens[used]].double()).sum(1)
        return gathered, y, gz, gweights.view(-1, topk), gx
    # the rows between the products are kept in the 16-bit type
    dtype = _DTYPES[case["dtype"]]
    a = _exact_rows(gathered)
    down = torch.zeros_like(gathered)
    mid = torch.zeros(n_rows, 2 * case["inner"], dtype=torch.float64, device=dev)
    for e, run_ in enumerate(mine):
        at = slice(offsets[e], offsets[e] + len(run_))
        if run_:
            mid[at] = a[at] @ _exact_weight(s["w1"][e], s["sw1"][e]).t()
            gate, up = mid[at].to(dtype).double().chunk(2, dim=1)
            down[at] = _exact_rows(gate * torch.sigmoid(gate) * up) @ _exact_weight(s["w2"][e], s["sw2"][e]).t()
    y = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device=dev)
    y.index_add_(0, tokens[used], weights[used, None] * down[rows_t[used]].to(dtype).double())
    return mid, down, y
