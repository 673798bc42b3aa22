"""Products of int8 operands with one scale per token and one per output channel.

    w8a8_int8_matmul        C[m, n] = out(Bs[n] * (As[m] * sum_k A[m, k] B[n, k]) + bias[n])
    w8a8_int8_grouped_mm    the same with one B per group of rows

They are to int8 models what ``w8a8_block_fp8_matmul`` and ``scaled_grouped_mm`` are to FP8 ones (the reference has int8
products inside its expert layer only, src/flag_gems/fused/fused_moe.py:1198-1347).  The sums are whole numbers
held exactly in 32 bits, whatever the order they are added in; each is rounded to fp32 once, scaled there, joined by
the bias there, and rounded to the output type.
"""
import logging
from typing import Optional

import torch

from .. import _cabi

logger = logging.getLogger(__name__.replace("flaggems_b200", "flag_gems", 1))

# Sums of more products of int8 values may leave 32 bits (2^14 each).
MAX_K = 131071


def _check_operands(a, b, k, k_b, output_dtype):
    assert k == k_b, f"A has {k} values per row, B {k_b}"
    if a.dtype != torch.int8 or b.dtype != torch.int8:
        raise NotImplementedError(f"operands must be int8, got {a.dtype} and {b.dtype}")
    if output_dtype not in _cabi.DTYPE_CODE:
        raise NotImplementedError(f"unsupported output dtype {output_dtype}")
    if k == 0 or k % 16 != 0 or k > MAX_K:
        raise NotImplementedError(f"K = {k} must be a positive multiple of 16, at most {MAX_K}")


def _scale(scale, shapes, name):
    """A scale of one of ``shapes``, or a single value, as contiguous fp32."""
    assert scale.numel() == 1 or tuple(scale.shape) in shapes, f"{name} must be a single value or one of the shapes {shapes}"
    return scale.float().contiguous()


def _rows_of_16_bytes(t):
    """[rows, K] with K contiguous and rows on 16-byte boundaries, copied only if it is not so already."""
    if (t.shape[-1] > 1 and t.stride(-1) != 1) or t.stride(-2) % 16 != 0 or t.stride(-2) < t.shape[-1] or t.data_ptr() % 16 != 0:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def w8a8_int8_matmul(
    A: torch.Tensor,
    B: torch.Tensor,
    As: torch.Tensor,
    Bs: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    output_dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """``A`` int8 [..., K], ``B`` int8 [N, K] (a linear layer's weight); K a multiple of 16.

    ``As`` float32: one value, or one per row ([...] or [..., 1]); ``Bs`` float32: one value, or one per
    output channel ([N] or [N, 1]); ``bias`` [N] in bf16, fp16 or fp32.  Returns [..., N] of ``output_dtype``
    (bf16, fp16 or fp32).  The scales that ``per_token_quant_int8`` returns fit as they are.  For inference: scales
    and bias that require a gradient are refused where one would be recorded.
    """
    logger.debug("GEMS W8A8_INT8_MATMUL")
    if A.is_cuda:
        c = _cabi.host.int8_mm(A, B, As, Bs, bias, output_dtype)
        if c is not None:
            return c
    assert A.dim() >= 1 and B.dim() == 2, "A must be [..., K] and B [N, K]"
    k = A.shape[-1]
    n = B.shape[0]
    _check_operands(A, B, k, B.shape[1], output_dtype)
    _cabi.refuse_gradients(As=As, Bs=Bs, bias=bias)
    lead = tuple(A.shape[:-1])
    As = _scale(As, (lead, lead + (1,)), "As")
    Bs = _scale(Bs, ((n,), (n, 1)), "Bs")
    if bias is not None:
        assert bias.shape == (n,), f"bias must have shape ({n},)"
        if bias.dtype not in _cabi.DTYPE_CODE:
            raise NotImplementedError(f"unsupported bias dtype {bias.dtype}")
        bias = bias.contiguous()
    _cabi.require_cuda(A, B, As, Bs, bias)
    _same_device(A, B, As, Bs, bias)
    c = A.new_empty(lead + (n,), dtype=output_dtype)
    if c.numel() == 0:
        return c
    A2, B = _rows_of_16_bytes(A.reshape(-1, k)), _rows_of_16_bytes(B)
    with _cabi.device_guard(A):
        _cabi.check(
            _cabi.lib().fg_scaled_mm_int8(
                _cabi.ptr(c), _cabi.ptr(A2), _cabi.ptr(B), _cabi.ptr(As), _cabi.ptr(Bs), _cabi.ptr(bias),
                0 if bias is None else _cabi.DTYPE_CODE[bias.dtype], A2.shape[0], n, k, A2.stride(0), B.stride(0), n,
                _cabi.SCALE_VECTOR if As.numel() > 1 else _cabi.SCALE_SCALAR,
                _cabi.SCALE_VECTOR if Bs.numel() > 1 else _cabi.SCALE_SCALAR,
                _cabi.DTYPE_CODE[output_dtype], 0, _cabi.stream_ptr(A.device),
            )
        )
    return c


def w8a8_int8_grouped_mm(
    A: torch.Tensor,
    B: torch.Tensor,
    As: torch.Tensor,
    Bs: torch.Tensor,
    offs: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    output_dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """Rows [offs[g - 1], offs[g]) of ``A`` int8 [M, K] times ``B[g]`` of ``B`` int8 [G, N, K]; K a multiple of 16.

    ``As`` float32, one value per row ([M] or [M, 1]); ``Bs`` float32 [G, N]; ``offs`` int32 [G], ascending, read on the
    device; ``bias`` [N] or [G, N], added in fp32.  Returns [M, N] of ``output_dtype``; rows from offs[-1] on
    belong to no group and are zeros.  ``moe_permute`` returns rows and ``offs`` that fit, ``per_token_quant_int8`` scales.
    For inference, as ``w8a8_int8_matmul``.
    """
    logger.debug("GEMS W8A8_INT8_GROUPED_MM")
    if A.is_cuda and bias is None:
        c = _cabi.host.int8_grouped_mm(A, B, As, Bs, offs, output_dtype)
        if c is not None:
            return c
    assert A.dim() == 2 and B.dim() == 3, "A must be [M, K] and B [G, N, K]"
    m, k = A.shape
    g, n, k_b = B.shape
    _check_operands(A, B, k, k_b, output_dtype)
    _cabi.refuse_gradients(As=As, Bs=Bs, bias=bias)
    assert tuple(As.shape) in ((m,), (m, 1)), f"As must have shape ({m},) or ({m}, 1)"
    assert tuple(Bs.shape) == (g, n), f"Bs must have shape ({g}, {n})"
    assert offs.shape == (g,) and offs.dtype == torch.int32, f"offs must be int32 of shape ({g},)"
    if bias is not None:
        assert tuple(bias.shape) in ((n,), (g, n)), f"bias must have shape ({n},) or ({g}, {n})"
        bias = bias.float().contiguous()
    _cabi.require_cuda(A, B, As, Bs, offs, bias)
    _same_device(A, B, As, Bs, offs, bias)
    c = torch.zeros((m, n), dtype=output_dtype, device=A.device) if g == 0 else A.new_empty((m, n), dtype=output_dtype)
    if c.numel() == 0 or g == 0:
        return c
    A = _rows_of_16_bytes(A)
    if not B.is_contiguous() or B.data_ptr() % 16 != 0:
        B = B.clone(memory_format=torch.contiguous_format)
    As, Bs, offs = As.float().contiguous(), Bs.float().contiguous(), offs.contiguous()
    L = _cabi.lib()
    with _cabi.device_guard(A):
        ws = torch.empty(int(L.fg_scaled_grouped_mm_workspace_bytes(m, g, k)) + 256, dtype=torch.uint8, device=A.device)
        _cabi.check(
            L.fg_scaled_grouped_mm_int8(
                _cabi.ptr(c), _cabi.ptr(A), _cabi.ptr(B), _cabi.ptr(As), _cabi.ptr(Bs), _cabi.ptr(bias),
                n if bias is not None and bias.dim() == 2 else 0, _cabi.ptr(offs), g, m, n, k, A.stride(0), n,
                _cabi.DTYPE_CODE[output_dtype], _cabi.ptr(ws), ws.numel(), _cabi.stream_ptr(A.device),
            )
        )
    return c


def _same_device(first, *others):
    for t in others:
        assert t is None or t.device == first.device, f"operands on {first.device} and {t.device}"
