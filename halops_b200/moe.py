"""Tokens in the order of the experts that a router gave them, and back: ``moe_sort``, ``moe_permute``,
``moe_permute_block_quant``, ``moe_unpermute`` and their gradients.  What stands around the grouped GEMMs of this package
(``group_block_gemm``, ``group_contiguous_gemm``), whose rows are in that order.  No counterpart in the reference.

A layer of experts on one device::

    order = moe_sort(topk_ids, num_experts)
    xq, xs = moe_permute_block_quant(x, order)
    group_block_gemm(xq, w13, xs, w13_sf, order.offsets, mid)
    hq, hs = swiglu_block_quant(mid, order.offsets)
    group_block_gemm(hq, w2, hs, w2_sf, order.offsets, down)
    y = moe_unpermute(down, order, topk_weights)

``group_contiguous_gemm`` wants runs that start on multiples of 64 rows and the expert of every row: ``moe_sort(ids, e,
align=64)``, ``group_wise_quant(moe_permute(x, order))`` and ``order.expert_ids``.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _native
from .gemm.block_scale import _IN_DTYPES, _OUT_DTYPES, _blocks, _check, _on_device, _pitch, _quant_outputs, _rows_ok

__all__ = ["MoeSort", "moe_permute", "moe_permute_backward", "moe_permute_block_quant", "moe_sort", "moe_unpermute",
           "moe_unpermute_backward"]

MAX_EXPERTS = 1024
MAX_PAIRS = 2**31 - 8192


class MoeSort(NamedTuple):
    """Where the pairs (token, slot) of a router's choice are in expert order; int32 CUDA tensors.  Those of one call may share a storage,
    which lives as long as the last of them (clone what is kept or saved alone)."""

    rows: torch.Tensor  # [tokens, topk]: the pair's row, -1 where its expert is not here
    pairs: torch.Tensor  # [n_rows]: token * topk + slot of the row, -1 where there is none
    offsets: torch.Tensor  # [num_experts + 1]: first row of each expert's run, and the end of the last
    expert_ids: torch.Tensor  # [n_rows]: the run that the row is in, num_experts - 1 behind the last
    align: int  # runs start on multiples of it


def moe_sort(topk_ids: torch.Tensor, num_experts: int, align: int = 1, use_pdl: bool = True) -> MoeSort:
    """Sorts the pairs (token, slot) of a router's choice by expert; pairs of one expert stay in their order.

    Args:
        topk_ids: [tokens, topk] contiguous CUDA tensor, int32 or int64, at most 2^31 - 8192 pairs.  Ids outside of [0, num_experts) are dropped (experts of another
            device: subtract the first one that is here).  A token may name an expert more than once.
        num_experts: experts here, at most 1024.
        align: every run starts on a multiple of it, at most 4096; the rows that pad a run have no pair.
        use_pdl: launch with programmatic stream serialisation.

    Returns:
        ``MoeSort``; its ``n_rows`` holds for any ids of this shape: all pairs, and ``align - 1`` rows more for each
        expert that can have one.
    """
    result = (_native.fast_path or _native.load_fast_path()).moe_sort(topk_ids, num_experts, align, use_pdl)
    if result is not None:
        return MoeSort(*result, align)
    _check(topk_ids.dim() == 2, "topk_ids must be a 2D tensor of shape [tokens, topk]")
    _check(topk_ids.dtype in (torch.int32, torch.int64), "topk_ids must be int32 or int64")
    _check(1 <= num_experts <= MAX_EXPERTS, f"num_experts must be in [1, {MAX_EXPERTS}], got {num_experts}")
    _check(1 <= align <= 4096, f"align must be in [1, 4096], got {align}")
    _check(topk_ids.is_contiguous(), "topk_ids must be contiguous")
    n = topk_ids.numel()
    _check(n <= MAX_PAIRS, f"at most 2^31 - 8192 pairs, got {n}")
    _on_device(topk_ids.device, topk_ids=topk_ids)
    n_rows = (n + min(num_experts, n) * (align - 1)) // align * align
    _check(n_rows < 2**31, f"at most 2^31 - 1 rows, got {n_rows}")
    rows, pairs, offsets, expert_ids = (torch.empty(shape, dtype=torch.int32, device=topk_ids.device)
                                        for shape in (tuple(topk_ids.shape), (n_rows,), (num_experts + 1,), (n_rows,)))
    _native.call("hq_moe_sort", topk_ids.data_ptr(), topk_ids.element_size(), topk_ids.size(0), topk_ids.size(1), num_experts, align, n_rows,
                 int(bool(use_pdl)), rows.data_ptr(), pairs.data_ptr(), offsets.data_ptr(), expert_ids.data_ptr(),
                 topk_ids.device.index, _native.current_stream(topk_ids.device))
    return MoeSort(rows, pairs, offsets, expert_ids, align)


def _order(sort: MoeSort, device) -> Tuple[int, int, int, int]:
    """(tokens, topk, rows, experts) of a sort whose tensors are what ``moe_sort`` returns."""
    for name, dim in (("rows", 2), ("pairs", 1), ("offsets", 1)):
        t = getattr(sort, name)
        _check(t.dim() == dim and t.dtype == torch.int32 and t.is_contiguous(), f"sort.{name} must be a contiguous int32 tensor as moe_sort returns it")
    _on_device(device, **{"sort.rows": sort.rows, "sort.pairs": sort.pairs, "sort.offsets": sort.offsets})
    _check(sort.offsets.size(0) >= 1, "sort.offsets must have num_experts + 1 elements")
    return sort.rows.size(0), sort.rows.size(1), sort.pairs.size(0), sort.offsets.size(0) - 1


def _rows_output(output, name, n_rows, h, like):
    if output is None:
        return torch.empty((n_rows, h), dtype=like.dtype, device=like.device)
    _check(output.is_contiguous() and output.dtype == like.dtype and tuple(output.shape) == (n_rows, h) and output.device == like.device,
           f"{name} must be a contiguous {like.dtype} tensor of shape [{n_rows}, {h}]")
    return output


def moe_permute(input: torch.Tensor, sort: MoeSort, output: Optional[torch.Tensor] = None, use_pdl: bool = True) -> torch.Tensor:
    """Every token's row once for each of its experts, in expert order.

    Args:
        input: [tokens, h] CUDA tensor of any type of 1, 2 or 4 bytes; rows may be strided.
        sort: what ``moe_sort`` returned for these tokens.
        output: optional contiguous [n_rows, h], returned as it is.
        use_pdl: launch with programmatic stream serialisation.

    Returns:
        [n_rows, h]; rows that pad a run are zero, rows from ``sort.offsets[-1]`` on are not written.
    """
    result = (_native.fast_path or _native.load_fast_path()).moe_permute(input, sort, output, use_pdl)
    if result is not None:
        return result
    _check(input.dim() == 2, "input must be a 2D tensor of shape [tokens, h]")
    _check(input.element_size() in (1, 2, 4), f"input must have elements of 1, 2 or 4 bytes, got {input.dtype}")
    _check(input.stride(1) == 1 or input.size(1) <= 1, "input rows must be contiguous")
    tokens, topk, n_rows, experts = _order(sort, input.device)
    _check(input.size(0) == tokens, f"input must have the sort's {tokens} tokens, got {input.size(0)}")
    out = _rows_output(output, "output", n_rows, input.size(1), input)
    _on_device(input.device, input=input)
    size = input.element_size()
    _native.call("hq_moe_permute", input.data_ptr(), input.stride(0) * size, tokens, input.size(1) * size, topk, sort.rows.data_ptr(),
                 sort.pairs.data_ptr(), sort.offsets.data_ptr(), experts, n_rows, int(sort.align > 1), int(bool(use_pdl)),
                 out.data_ptr(), input.device.index, _native.current_stream(input.device))
    return out


def moe_permute_block_quant(
    input: torch.Tensor,
    sort: MoeSort,
    use_pdl: bool = True,
    output_quant: Optional[torch.Tensor] = None,
    output_sf: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``block_quant(moe_permute(input, sort))`` in one pass: every token is read and quantised once.

    Args:
        input: [tokens, h] CUDA tensor, bfloat16 or float16, ``h`` a multiple of 16; rows may be strided (16-byte aligned).
        sort / use_pdl: as for ``moe_permute``.
        output_quant / output_sf: optional contiguous outputs, returned as they are.

    Returns:
        [n_rows, h] float8_e4m3fn and [n_rows, ceil(h/128)] float32; rows from ``sort.offsets[-1]`` on are not written.
    """
    result = (_native.fast_path or _native.load_fast_path()).moe_permute_block_quant(input, sort, use_pdl, output_quant, output_sf)
    if result is not None:
        return result
    _check(input.dim() == 2, "input must be a 2D tensor of shape [tokens, h]")
    _check(input.dtype in _IN_DTYPES, "input dtype must be bfloat16 or float16")
    h = input.size(1)
    _check(h % 16 == 0, f"hidden size must be divisible by 16, got {h}")
    _check(_rows_ok(input), "input rows must be contiguous and 16-byte aligned")
    tokens, topk, n_rows, experts = _order(sort, input.device)
    _check(input.size(0) == tokens, f"input must have the sort's {tokens} tokens, got {input.size(0)}")
    q, sf = _quant_outputs(output_quant, output_sf, (n_rows, h), (n_rows, _blocks(h)), input.device)
    _on_device(input.device, input=input)
    _native.call("hq_moe_permute_block_quant", input.data_ptr(), _pitch(input), _IN_DTYPES[input.dtype], tokens, h, topk,
                 sort.rows.data_ptr(), sort.pairs.data_ptr(), sort.offsets.data_ptr(), experts, n_rows, int(sort.align > 1),
                 int(bool(use_pdl)), q.data_ptr(), sf.data_ptr(), input.device.index, _native.current_stream(input.device))
    return q, sf


def _tokens_input(input, sort, weights, name="input"):
    _check(input.dim() == 2, f"{name} must be a 2D tensor of shape [n_rows, h]")
    _check(input.dtype in _OUT_DTYPES, f"{name} dtype must be bfloat16, float16 or float32")
    _check(input.stride(1) == 1 or input.size(1) <= 1, f"{name} rows must be contiguous")
    tokens, topk, n_rows, experts = _order(sort, input.device)
    _check(input.size(0) == n_rows, f"{name} must have the sort's {n_rows} rows, got {input.size(0)}")
    _check(weights is None or (weights.dtype == torch.float32 and tuple(weights.shape) == (tokens, topk) and weights.is_contiguous()),
           f"weights must be a contiguous float32 tensor of shape [{tokens}, {topk}]")
    _on_device(input.device, weights=weights, **{name: input})
    return tokens, topk, n_rows, experts


def moe_unpermute(input: torch.Tensor, sort: MoeSort, weights: Optional[torch.Tensor] = None, use_pdl: bool = True) -> torch.Tensor:
    """Back to the tokens: ``out[t] = sum over slots of weights[t, slot] * input[sort.rows[t, slot]]`` in float32, in the order of the
    slots, rounded once.  Slots without a row are left out, their weight is not read into the sum; a token without any row
    is zero.

    Args:
        input: [n_rows, h] bfloat16, float16 or float32; rows may be strided.
        sort: what ``moe_sort`` returned.
        weights: float32 [tokens, topk], or None for ones.
        use_pdl: launch with programmatic stream serialisation.

    Returns:
        [tokens, h] of the input's type.
    """
    result = (_native.fast_path or _native.load_fast_path()).moe_unpermute(input, sort, weights, use_pdl)
    if result is not None:
        return result
    tokens, topk, n_rows, _ = _tokens_input(input, sort, weights)
    out = torch.empty((tokens, input.size(1)), dtype=input.dtype, device=input.device)
    _native.call("hq_moe_unpermute", input.data_ptr(), input.stride(0), _OUT_DTYPES[input.dtype], n_rows, input.size(1), tokens, topk,
                 sort.rows.data_ptr(), None if weights is None else weights.data_ptr(), int(bool(use_pdl)), out.data_ptr(),
                 input.device.index, _native.current_stream(input.device))
    return out


def moe_permute_backward(grad_output: torch.Tensor, sort: MoeSort, use_pdl: bool = True) -> torch.Tensor:
    """The gradient of ``moe_permute``: every token's sum, in float32, of its rows of ``grad_output`` [n_rows, h]."""
    return moe_unpermute(grad_output, sort, None, use_pdl)


def moe_unpermute_backward(
    grad_output: torch.Tensor,
    input: torch.Tensor,
    sort: MoeSort,
    weights: Optional[torch.Tensor] = None,
    use_pdl: bool = True,
    grad_input: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The gradients of ``moe_unpermute(input, sort, weights)``.

    Args:
        grad_output: [tokens, h], of the input's type; rows may be strided.
        input / sort / weights: as they were given to ``moe_unpermute``.
        use_pdl: launch with programmatic stream serialisation.
        grad_input: optional contiguous [n_rows, h], returned as it is.

    Returns:
        ``(grad_input, grad_weights)``: [n_rows, h] with ``weights[pair] * grad_output[token]`` (rows that pad a run are zero, rows
        from ``sort.offsets[-1]`` on are not written), and float32 [tokens, topk] with the products
        ``<grad_output[token], input[row]>`` (0 for a slot without a row), None where ``weights`` is.  A product is summed by a warp, or
        by 256 threads where there are few pairs, in pieces whose size goes by the rows' alignment: the same call gives the same bits, the
        same token in a batch of another size may differ in the last ones.
    """
    result = (_native.fast_path or _native.load_fast_path()).moe_unpermute_backward(grad_output, input, sort, weights, use_pdl, grad_input)
    if result is not None:
        return result
    tokens, topk, n_rows, experts = _tokens_input(input, sort, weights)
    _check(grad_output.dim() == 2 and tuple(grad_output.shape) == (tokens, input.size(1)) and grad_output.dtype == input.dtype,
           f"grad_output must be a {input.dtype} tensor of shape [{tokens}, {input.size(1)}]")
    _check(grad_output.stride(1) == 1 or input.size(1) <= 1, "grad_output rows must be contiguous")
    gz = _rows_output(grad_input, "grad_input", n_rows, input.size(1), input)
    gw = None if weights is None else torch.empty_like(weights)
    _on_device(input.device, grad_output=grad_output)
    _native.call("hq_moe_unpermute_backward", grad_output.data_ptr(), grad_output.stride(0), input.data_ptr(), input.stride(0),
                 _OUT_DTYPES[input.dtype], n_rows, input.size(1), tokens, topk, sort.rows.data_ptr(), sort.pairs.data_ptr(),
                 sort.offsets.data_ptr(), experts, int(sort.align > 1), None if weights is None else weights.data_ptr(),
                 int(bool(use_pdl)), gz.data_ptr(), None if gw is None else gw.data_ptr(), input.device.index,
                 _native.current_stream(input.device))
    return gz, gw
