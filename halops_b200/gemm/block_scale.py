"""FP8 products whose operands carry a float32 scale per block of 128: ``block_quant``, ``swiglu_block_quant``,
``block_gemm`` and ``group_block_gemm``.  Checkpoints keep weights in this form (a scale per 128 x 128) and
activations are quantised to it on the way (a scale per 128 values of a row); the block scales of the MX kinds of this
package (``group_wise_quant``, ``dense_gemm``) are powers of two per 32 values and cannot hold them.  No counterpart in
the reference.

Training: with ``w`` [N, K] in blocks of 128 x 128, the gradient of the input is a product with the transposed weight
(``block_quant(w, (128, 128), transpose=True)``, or the transposed codes and scales), the gradient of the weight one of the
two transposed operands (``block_quant(grad, transpose=True)``, ``block_quant(x, transpose=True)``) with a scale per
row on both sides::

    gq, gs = block_quant(grad)                          # [M, N]
    block_gemm(gq, wt, gs, wts, grad_x)                 # wt [K, N], wts [K/128, N/128]
    gtq, gts = block_quant(grad, transpose=True)        # [N, M16]
    xtq, xts = block_quant(x, transpose=True)           # [K, M16]
    block_gemm(gtq, xtq, gts, xts, grad_w)              # [N, K] float32
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _native

__all__ = ["block_gemm", "block_quant", "group_block_gemm", "swiglu_block_quant"]

BLOCK = 128
_IN_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_OUT_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _on_device(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        _check(t is None or t.is_cuda, f"{name} must be a CUDA tensor (this library has no CPU path)")
        _check(t is None or t.device == device, f"{name} must be on the input's device, got {getattr(t, 'device', None)}")


def _rows_ok(t: torch.Tensor) -> bool:
    """16-bit rows that the kernels can read: contiguous, on 16 bytes."""
    return (t.stride(-1) == 1 and t.data_ptr() % 16 == 0
            and all(s % 8 == 0 or n <= 1 for s, n in zip(t.stride()[:-1], t.shape[:-1])))


def _pitch(t: torch.Tensor, dim: int = -2) -> int:
    """Elements between rows (of a single row: of no consequence, whatever its stride)."""
    return t.stride(dim) if t.size(dim) > 1 else (t.size(-1) + 7) // 8 * 8


def _quant_outputs(q, sf, q_shape, sf_shape, device):
    if q is None:
        q = torch.empty(q_shape, dtype=torch.float8_e4m3fn, device=device)
    else:
        _check(q.is_contiguous() and q.dtype == torch.float8_e4m3fn and tuple(q.shape) == tuple(q_shape) and q.device == device,
               f"output_quant must be a contiguous float8_e4m3fn tensor of shape {list(q_shape)}")
    if sf is None:
        sf = torch.empty(sf_shape, dtype=torch.float32, device=device)
    else:
        _check(sf.is_contiguous() and sf.dtype == torch.float32 and tuple(sf.shape) == tuple(sf_shape) and sf.device == device,
               f"output_sf must be a contiguous float32 tensor of shape {list(sf_shape)}")
    return q, sf


def block_quant(
    input: torch.Tensor,
    block: Tuple[int, int] = (1, 128),
    transpose: bool = False,
    use_pdl: bool = True,
    output_quant: Optional[torch.Tensor] = None,
    output_sf: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """BF16/FP16 to e4m3 with a float32 scale per block: ``scale = max(max |x|, 1e-10) / 448``, codes nearest to
    ``x / scale``, ties to even.  A NaN or an infinity makes its block's scale NaN or infinite.

    Args:
        input: [m, k] CUDA tensor, bfloat16 or float16, ``k`` a multiple of 16; rows may be strided (16-byte aligned).
            Blocks of (128, 128) are also taken of [e, m, k].
        block: (1, 128), for activations and gradients, or (128, 128), for weights.
        transpose: quantise the transposed matrix and return it as such; blocks of (1, 128) then lie along ``m``.
        use_pdl: launch with programmatic stream serialisation.
        output_quant / output_sf: optional contiguous outputs, returned as they are.

    Returns:
        ``(output_quant, output_sf)``.  Without ``transpose`` [.., m, k] float8_e4m3fn and float32 [m, ceil(k/128)] or
        [.., ceil(m/128), ceil(k/128)]; with it [.., k, m rounded up to 16] (columns from ``m`` on are zero, so that it can be an
        operand of ``block_gemm``) and [k, ceil(m/128)] or [.., ceil(k/128), ceil(m/128)].
    """
    result = (_native.fast_path or _native.load_fast_path()).block_quant(input, block, transpose, use_pdl, output_quant, output_sf)
    if result is not None:
        return result
    block = tuple(block)
    _check(block in ((1, 128), (128, 128)), f"block must be (1, 128) or (128, 128), got {block}")
    square = block == (128, 128)
    _check(input.dim() == 2 or (square and input.dim() == 3),
           "input must be a 2D tensor of shape [m, k] (or [e, m, k] for blocks of (128, 128))")
    _check(input.dtype in _IN_DTYPES, "input dtype must be bfloat16 or float16")
    m, k = input.shape[-2:]
    _check(k % 16 == 0, f"k must be divisible by 16, got k={k}")
    _check(_rows_ok(input), "input rows must be contiguous and 16-byte aligned")
    lead = tuple(input.shape[:-2])
    q_shape = lead + ((k, (m + 15) // 16 * 16) if transpose else (m, k))
    rows, cols = (k, m) if transpose else (m, k)
    sf_shape = lead + (_blocks(rows) if square else rows, _blocks(cols))
    q, sf = _quant_outputs(output_quant, output_sf, q_shape, sf_shape, input.device)
    _on_device(input.device, input=input)
    _native.call(
        "hq_block_quant", input.data_ptr(), _pitch(input), _pitch(input, 0) if input.dim() == 3 else 0, _IN_DTYPES[input.dtype],
        input.size(0) if input.dim() == 3 else 1, m, k, block[0], int(bool(transpose)), int(bool(use_pdl)), q.data_ptr(),
        sf.data_ptr(), input.device.index, _native.current_stream(input.device))
    return q, sf


def swiglu_block_quant(
    input: torch.Tensor,
    offsets: Optional[torch.Tensor] = None,
    use_pdl: bool = True,
    output_quant: Optional[torch.Tensor] = None,
    output_sf: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``silu(gate) * up`` of rows ``[gate | up]``, in float32 (off by less than 2^-20 of its value, for any gate whose product is a
    normal number), quantised in blocks of (1, 128) as ``block_quant`` does: what comes between the two products of a gated MLP or of
    an expert.

    Args:
        input: [m, 2k] CUDA tensor, bfloat16 or float16, ``k`` a multiple of 16; rows may be strided (16-byte aligned).
        offsets: optional int32 CUDA tensor of row numbers (``MoeSort.offsets``): rows from its last value on are
            neither read nor written.
        use_pdl / output_quant / output_sf: as for ``block_quant``.

    Returns:
        [m, k] float8_e4m3fn and [m, ceil(k/128)] float32.
    """
    result = (_native.fast_path or _native.load_fast_path()).swiglu_block_quant(input, offsets, use_pdl, output_quant, output_sf)
    if result is not None:
        return result
    _check(input.dim() == 2, "input must be a 2D tensor of shape [m, 2k]")
    _check(input.dtype in _IN_DTYPES, "input dtype must be bfloat16 or float16")
    m, k = input.size(0), input.size(1) // 2
    _check(input.size(1) % 32 == 0, f"half of the columns must be divisible by 16, got {input.size(1)} columns")
    _check(_rows_ok(input), "input rows must be contiguous and 16-byte aligned")
    _check(offsets is None or (offsets.dim() == 1 and offsets.size(0) > 0 and offsets.dtype == torch.int32 and offsets.is_contiguous()),
           "offsets must be a contiguous 1D int32 tensor")
    q, sf = _quant_outputs(output_quant, output_sf, (m, k), (m, _blocks(k)), input.device)
    _on_device(input.device, input=input, offsets=offsets)
    limit = None if offsets is None else offsets.data_ptr() + 4 * (offsets.size(0) - 1)
    _native.call(
        "hq_swiglu_block_quant", input.data_ptr(), _pitch(input), _IN_DTYPES[input.dtype], m, k, limit, int(bool(use_pdl)),
        q.data_ptr(), sf.data_ptr(), input.device.index, _native.current_stream(input.device))
    return q, sf


def _operands(input, weight, sfa, sfb, output, n):
    k = input.size(1)
    _check(input.dtype == torch.float8_e4m3fn and weight.dtype == torch.float8_e4m3fn, "input and weight must be float8_e4m3fn tensors")
    _check(weight.size(-1) == k, f"input K must match weight K, got input K={k}, weight K={weight.size(-1)}")
    _check(k >= 16 and k % 16 == 0, f"K must be a positive multiple of 16, got K={k}")
    _check(sfa.dtype == torch.float32 and sfb.dtype == torch.float32, "sfa and sfb must be float32 tensors")
    _check(tuple(sfa.shape) == (input.size(0), _blocks(k)), f"sfa must be [{input.size(0)}, {_blocks(k)}], got {list(sfa.shape)}")
    _check(output.dim() == 2 and output.size(0) == input.size(0) and output.size(1) == n,
           f"output must be [{input.size(0)}, {n}], got {list(output.shape)}")
    _check(output.dtype in _OUT_DTYPES, "output dtype must be bfloat16, float16 or float32")
    _check(input.is_contiguous() and weight.is_contiguous() and sfa.is_contiguous() and sfb.is_contiguous(),
           "input, weight, sfa and sfb must be contiguous")
    _check((output.stride(1) == 1 or n <= 1) and (output.stride(0) >= n or input.size(0) <= 1), "output rows must be contiguous")
    _check(input.data_ptr() % 16 == 0 and weight.data_ptr() % 16 == 0, "input and weight must be 16-byte aligned")
    _on_device(input.device, input=input, weight=weight, sfa=sfa, sfb=sfb, output=output)
    return k


def block_gemm(
    input: torch.Tensor,
    weight: torch.Tensor,
    sfa: torch.Tensor,
    sfb: torch.Tensor,
    output: torch.Tensor,
    sm_count: int = -1,
    use_pdl: bool = True,
) -> None:
    """``output = (input * sfa) @ (weight * sfb)^T``, summed in float32 and rounded once.  The two scales of a block are multiplied in float32 (with
    a scale per row on both sides one after the other onto the sums): their product has to be a finite, normal number, as those of
    ``block_quant`` are for values whose magnitudes multiply to less than 1e43.

    Args:
        input: [M, K] float8_e4m3fn, ``K`` a positive multiple of 16.
        weight: [N, K] float8_e4m3fn.
        sfa: float32 [M, ceil(K/128)], as ``block_quant(x)`` returns it.
        sfb: float32 [ceil(N/128), ceil(K/128)] (``block_quant(w, (128, 128))``) or [N, ceil(K/128)], a scale per row of
            ``weight`` (``block_quant(w)``).  With ``N == 1`` the two are the same.
        output: [M, N] bfloat16, float16 or float32, written in place; rows may be strided.
        sm_count: SMs to use, -1 for all.
        use_pdl: launch with programmatic stream serialisation.
    """
    if (_native.fast_path or _native.load_fast_path()).block_gemm(input, weight, sfa, sfb, None, output, sm_count, use_pdl):
        return
    _check(input.dim() == 2, "input must be a 2D tensor of shape [M, K]")
    _check(weight.dim() == 2, "weight must be a 2D tensor of shape [N, K]")
    m, n = input.size(0), weight.size(0)
    k = _operands(input, weight, sfa, sfb, output, n)
    square = tuple(sfb.shape) == (_blocks(n), _blocks(k))
    _check(square or tuple(sfb.shape) == (n, _blocks(k)),
           f"sfb must be [{_blocks(n)}, {_blocks(k)}] (per 128 x 128) or [{n}, {_blocks(k)}] (per row), got {list(sfb.shape)}")
    if m == 0 or n == 0:
        return
    _native.call(
        "hq_block_gemm", input.data_ptr(), weight.data_ptr(), sfa.data_ptr(), sfb.data_ptr(), output.data_ptr(),
        _OUT_DTYPES[output.dtype], m, n, k, int(not square), max(output.stride(0), n), int(sm_count), int(bool(use_pdl)), input.device.index,
        _native.current_stream(input.device))


def group_block_gemm(
    input: torch.Tensor,
    weight: torch.Tensor,
    sfa: torch.Tensor,
    sfb: torch.Tensor,
    offsets: torch.Tensor,
    output: torch.Tensor,
    sm_count: int = -1,
    use_pdl: bool = True,
) -> None:
    """``block_gemm`` for rows in runs of one expert each: rows ``offsets[e] .. offsets[e + 1]`` are multiplied by
    ``weight[e]``; rows outside of all runs are not written.

    Args:
        input: [M, K] float8_e4m3fn, rows in expert order (``moe_permute_block_quant``).
        weight: [num_experts, N, K] float8_e4m3fn, at most 1024 experts.
        sfa: float32 [M, ceil(K/128)].
        sfb: float32 [num_experts, ceil(N/128), ceil(K/128)].
        offsets: int32 [num_experts + 1], non-decreasing (``MoeSort.offsets``); runs may start on any row and be empty.
        output: [M, N] bfloat16, float16 or float32, written in place; rows may be strided.
        sm_count / use_pdl: as for ``block_gemm``.
    """
    if (_native.fast_path or _native.load_fast_path()).block_gemm(input, weight, sfa, sfb, offsets, output, sm_count, use_pdl):
        return
    _check(input.dim() == 2, "input must be a 2D tensor of shape [M, K]")
    _check(weight.dim() == 3, "weight must be a 3D tensor of shape [num_experts, N, K]")
    m, n, experts = input.size(0), weight.size(1), weight.size(0)
    k = _operands(input, weight, sfa, sfb, output, n)
    _check(tuple(sfb.shape) == (experts, _blocks(n), _blocks(k)),
           f"sfb must be [{experts}, {_blocks(n)}, {_blocks(k)}], got {list(sfb.shape)}")
    _check(offsets.dim() == 1 and offsets.dtype == torch.int32 and offsets.size(0) == experts + 1 and offsets.is_contiguous(),
           f"offsets must be a contiguous int32 tensor of {experts + 1} elements")
    _on_device(input.device, offsets=offsets)
    if m == 0 or n == 0 or experts == 0:
        return
    _native.call(
        "hq_group_block_gemm", input.data_ptr(), weight.data_ptr(), sfa.data_ptr(), sfb.data_ptr(), offsets.data_ptr(), output.data_ptr(),
        _OUT_DTYPES[output.dtype], experts, m, n, k, max(output.stride(0), n), int(sm_count), int(bool(use_pdl)), input.device.index,
        _native.current_stream(input.device))
