"""Refusals of the block-128 and expert-order entry points, without a device: the C ABI's and the Python wrappers'."""

import ctypes

import pytest
import torch

import halops_b200 as hq
from test_kernel_waits_cpu import test_roles_read_the_abort_flag_as_whole_warps as read_abort_flag
from test_kernel_waits_cpu import test_roles_wait_as_whole_warps as wait_as_warps

P = ctypes.cast(256, ctypes.c_void_p)  # a pointer that a refusal must not follow
ODD = ctypes.cast(264, ctypes.c_void_p)


@pytest.fixture(scope="module")
def call():
    from halops_b200 import _native, build

    build.build()

    def run(name, *args):
        err = ctypes.create_string_buffer(512)
        rc = getattr(_native.lib(), name)(*args, err, 512)
        return rc, err.value.decode()

    return run


def _quant(call, x=P, ld=256, batch=0, dtype=0, e=1, m=4, k=256, rows=1, t=0, q=P, sf=P):
    return call("hq_block_quant", x, ld, batch, dtype, e, m, k, rows, t, 0, q, sf, 0, None)


@pytest.mark.parametrize("args,text", [
    (dict(dtype=2), "bfloat16 or float16"), (dict(rows=64), r"block must be"), (dict(k=250), "divisible by 16, got k=250"),
    (dict(m=-1), "too large"), (dict(k=1 << 23), "too large"), (dict(e=70000, rows=128), "too large"), (dict(e=2), r"blocks of \(1, 128\)"),
    (dict(x=None), "null pointer"), (dict(q=None), "null pointer"), (dict(ld=128), "16-byte aligned"), (dict(ld=260), "16-byte aligned"),
    (dict(x=ODD), "16-byte aligned"), (dict(e=2, rows=128, batch=1020), "16-byte aligned"), (dict(q=ODD), "output_quant"),
    (dict(m=1 << 31, k=1 << 20, ld=1 << 20), "too large for one launch"),
])
def test_block_quant(call, args, text):
    rc, msg = _quant(call, **args)
    import re

    assert rc == 1 and re.search(text, msg), msg


def test_nothing_to_do_is_no_error(call):
    assert _quant(call, m=0, x=None, q=None, sf=None)[0] == 0
    assert _quant(call, k=0, x=None)[0] == 0
    assert call("hq_swiglu_block_quant", None, 0, 0, 0, 128, None, 0, None, None, 0, None)[0] == 0
    assert call("hq_block_gemm", None, None, None, None, None, 0, 0, 128, 128, 0, 128, -1, 0, 0, None)[0] == 0
    assert call("hq_group_block_gemm", None, None, None, None, None, None, 0, 4, 0, 128, 128, 128, -1, 0, 0, None)[0] == 0
    assert call("hq_moe_permute", None, 0, 0, 64, 2, None, None, None, 4, 0, 1, 0, None, 0, None)[0] == 0
    assert call("hq_moe_permute_block_quant", None, 0, 0, 0, 64, 2, None, None, None, 4, 0, 1, 0, None, None, 0, None)[0] == 0
    assert call("hq_moe_unpermute", None, 0, 0, 0, 64, 0, 2, None, None, 0, None, 0, None)[0] == 0
    assert call("hq_moe_unpermute_backward", None, 0, None, 0, 0, 0, 64, 0, 2, None, None, None, 4, 0, None, 0, None, None, 0, None)[0] == 0


def test_swiglu(call):
    def run(x=P, ld=512, dtype=0, m=4, k=256, q=P, sf=P):
        return call("hq_swiglu_block_quant", x, ld, dtype, m, k, None, 0, q, sf, 0, None)

    for args, text in ((dict(dtype=2), "bfloat16 or float16"), (dict(k=100), "divisible by 16"), (dict(ld=256), "16-byte aligned"),
                       (dict(x=None), "null pointer"), (dict(sf=None), "null pointer"), (dict(m=-2), "too large")):
        rc, msg = run(**args)
        assert rc == 1 and text in msg, msg


def test_products(call):
    def dense(a=P, b=P, sfa=P, sfb=P, out=P, dtype=0, m=8, n=128, k=256, ldo=128):
        return call("hq_block_gemm", a, b, sfa, sfb, out, dtype, m, n, k, 0, ldo, -1, 0, 0, None)

    def group(offsets=P, e=4, m=8, n=128, k=256, dtype=0):
        return call("hq_group_block_gemm", P, P, P, P, offsets, P, dtype, e, m, n, k, n, -1, 0, 0, None)

    for args, text in ((dict(dtype=3), "output dtype"), (dict(k=0), "K must be a positive multiple of 16"), (dict(k=24), "got K=24"),
                       (dict(m=-1), "at most 2^31 - 256"), (dict(n=1 << 31), "at most 2^31 - 256"), (dict(a=None), "null pointer"),
                       (dict(a=ODD), "16-byte aligned"), (dict(ldo=100), "row stride of 100"),
                       (dict(m=1 << 30, n=1 << 20, ldo=1 << 20), "too many tiles")):
        rc, msg = dense(**args)
        assert rc == 1 and text in msg, msg
    for args, text in ((dict(offsets=None), "null pointer"), (dict(e=1025), "at most 1024 experts"), (dict(e=1000, n=1 << 22), "weight rows"),
                       (dict(k=8), "got K=8")):
        rc, msg = group(**args)
        assert rc == 1 and text in msg, msg


def test_moe(call):
    def sort(size=4, tokens=8, topk=2, experts=4, align=1, n_rows=16, ids=P):
        return call("hq_moe_sort", ids, size, tokens, topk, experts, align, n_rows, 0, P, P, P, P, 0, None)

    for args, text in ((dict(size=2), "int32 or int64"), (dict(experts=0), "at least 1"), (dict(experts=1025), "1024 experts"),
                       (dict(align=0), "align must be"), (dict(n_rows=15), "16 rows are needed"), (dict(align=64, n_rows=200), "256 rows are needed"),
                       (dict(tokens=1 << 30, topk=4), "at most 2^31 - 1 pairs"), (dict(ids=None), "null pointer")):
        rc, msg = sort(**args)
        assert rc == 1 and text in msg, msg
    rc, msg = call("hq_moe_permute", P, 64, 8, 1 << 25, 2, P, P, P, 4, 16, 0, 0, P, 0, None)
    assert rc == 1 and "16 MiB" in msg
    rc, msg = call("hq_moe_permute", P, 64, 8, 64, 2, None, P, P, 4, 16, 0, 0, P, 0, None)
    assert rc == 1 and "null pointer" in msg
    rc, msg = call("hq_moe_permute_block_quant", P, 64, 0, 8, 40, 2, P, P, P, 4, 16, 0, 0, P, P, 0, None)
    assert rc == 1 and "divisible by 16" in msg
    rc, msg = call("hq_moe_unpermute", P, 64, 5, 16, 64, 8, 2, P, P, 0, P, 0, None)
    assert rc == 1 and "bfloat16, float16 or float32" in msg
    rc, msg = call("hq_moe_unpermute_backward", P, 64, None, 64, 0, 16, 64, 8, 2, P, P, P, 4, 0, P, 0, P, P, 0, None)
    assert rc == 1 and "null pointer" in msg


def test_python_refusals_without_a_device():
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    f8 = lambda *s: torch.zeros(*s).to(torch.float8_e4m3fn)  # noqa: E731
    order = hq.MoeSort(torch.zeros(8, 2, dtype=torch.int32), torch.zeros(16, dtype=torch.int32), torch.zeros(5, dtype=torch.int32),
                       torch.zeros(16, dtype=torch.int32), 1)
    cases = [
        (lambda: hq.block_quant(bf(4, 256), (1, 64)), "block must be"),
        (lambda: hq.block_quant(bf(256)), "2D tensor"),
        (lambda: hq.block_quant(bf(2, 4, 256)), "2D tensor"),
        (lambda: hq.block_quant(torch.zeros(4, 256)), "bfloat16 or float16"),
        (lambda: hq.block_quant(bf(4, 100)), "divisible by 16, got k=100"),
        (lambda: hq.block_quant(bf(256, 4).t()), "16-byte aligned"),
        (lambda: hq.block_quant(bf(4, 256), output_sf=torch.zeros(4, 3)), r"output_sf must be a contiguous float32 tensor of shape \[4, 2\]"),
        (lambda: hq.block_quant(bf(4, 256), output_quant=bf(4, 256)), "output_quant must be"),
        (lambda: hq.block_quant(bf(4, 256)), "input must be a CUDA tensor"),
        (lambda: hq.swiglu_block_quant(bf(4, 80)), "divisible by 16, got 80"),
        (lambda: hq.swiglu_block_quant(bf(4, 64), torch.zeros(3)), "offsets must be"),
        (lambda: hq.swiglu_block_quant(bf(4, 64)), "CUDA tensor"),
        (lambda: hq.block_gemm(bf(4, 256), f8(8, 256), torch.zeros(4, 2), torch.zeros(1, 2), bf(4, 8)), "float8_e4m3fn"),
        (lambda: hq.block_gemm(f8(4, 256), f8(8, 128), torch.zeros(4, 2), torch.zeros(1, 2), bf(4, 8)), "input K=256, weight K=128"),
        (lambda: hq.block_gemm(f8(4, 250), f8(8, 250), torch.zeros(4, 2), torch.zeros(1, 2), bf(4, 8)), "multiple of 16, got K=250"),
        (lambda: hq.block_gemm(f8(4, 256), f8(8, 256), torch.zeros(4, 3), torch.zeros(1, 2), bf(4, 8)), r"sfa must be \[4, 2\]"),
        (lambda: hq.block_gemm(f8(4, 256), f8(8, 256), torch.zeros(4, 2), torch.zeros(1, 2), bf(4, 9)), r"output must be \[4, 8\]"),
        (lambda: hq.block_gemm(f8(4, 256), f8(8, 256), torch.zeros(4, 2), torch.zeros(1, 2), torch.zeros(4, 8).double()), "output dtype"),
        (lambda: hq.block_gemm(f8(4, 256), f8(8, 256), torch.zeros(4, 2), torch.zeros(1, 2), bf(4, 8)), "CUDA tensor"),
        (lambda: hq.group_block_gemm(f8(4, 256), f8(8, 256), torch.zeros(4, 2), torch.zeros(1, 2), None, bf(4, 8)), "3D tensor"),
        (lambda: hq.moe_sort(torch.zeros(4, dtype=torch.int32), 4), "2D tensor"),
        (lambda: hq.moe_sort(torch.zeros(4, 2), 4), "int32 or int64"),
        (lambda: hq.moe_sort(torch.zeros(4, 2, dtype=torch.int32), 0), r"num_experts must be in \[1, 1024\]"),
        (lambda: hq.moe_sort(torch.zeros(4, 2, dtype=torch.int32), 4, align=0), "align must be"),
        (lambda: hq.moe_sort(torch.zeros(4, 2, dtype=torch.int32), 4), "CUDA tensor"),
        (lambda: hq.moe_permute(bf(8, 32).double(), order), "1, 2 or 4 bytes"),
        (lambda: hq.moe_permute(bf(8, 32), order), "CUDA tensor"),
        (lambda: hq.moe_unpermute(f8(16, 32), order), "bfloat16, float16 or float32"),
        (lambda: hq.moe_unpermute_backward(bf(8, 32), bf(16, 32), order), "CUDA tensor"),
    ]
    for make, text in cases:
        with pytest.raises(RuntimeError, match=text):
            make()


def test_roles_of_the_block_kernel_wait_as_whole_warps():
    wait_as_warps("block_gemm.cu")
    read_abort_flag("block_gemm.cu")
    wait_as_warps("gemm_common.cuh")


def test_codes_of_the_rounded_quotient_are_those_of_the_exact_one():
    """The arithmetic of the kernels' code (x * fl(448 / amax), rounded to a multiple of 8 units) against the exact quotient, for every
    significand of a bf16 maximum with every significand of a bf16 value, and for random fp16 ones."""
    import numpy as np

    def kernel(x, amax):
        x, amax = x.astype(np.float32), amax.astype(np.float32)
        q = x * (np.float32(448) / amax)
        return ((q.view(np.uint32) + np.uint32(4)) & np.uint32(0xFFFFFFF8)).view(np.float32)

    def e4m3(v):
        v = v.astype(np.float64)
        step = np.exp2(np.maximum(np.frexp(v)[1] - 1, -6) - 3)
        return np.rint(v / step) * step

    def check(x, amax):
        exact = x.astype(np.float64) * 448 / amax.astype(np.float64)
        assert (e4m3(kernel(x, amax)) == e4m3(exact)).all()

    a = np.arange(128, 256)
    for shift in range(0, 20):
        x, amax = np.meshgrid(a * 2.0**-shift, a.astype(np.float64))
        keep = x <= amax
        check(x[keep], amax[keep])
    r = np.random.RandomState(0)
    x, amax = r.randint(1024, 2048, 1 << 20) * 2.0 ** -r.randint(0, 20, 1 << 20), r.randint(1024, 2048, 1 << 20).astype(np.float64)
    keep = x <= amax
    check(x[keep], amax[keep])
