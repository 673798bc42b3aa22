"""per_token_quant_int8: one scale per row, q = clamp(round_half_even(x / s), -128, 127), s = max(max|x|, 1e-10) / 127.

The arithmetic of the per-token branch of ``_int8_quantize`` (src/flag_gems/fused/fused_moe.py:732-739 of the
reference), as an operator of its own: what it returns are the operands of ``w8a8_int8_matmul`` and
``w8a8_int8_grouped_mm``.
"""
import logging
from typing import Tuple

import torch

from .. import _cabi

logger = logging.getLogger(__name__.replace("flaggems_b200", "flag_gems", 1))


def per_token_quant_int8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Quantise ``x`` [..., K] (bf16, fp16 or fp32) per row.

    Returns ``(q, s)``: ``q`` int8 with the shape of ``x`` and ``s`` float32 of shape ``x.shape[:-1] + (1,)``.
    Rows have to start on 16-byte boundaries and K has to be a multiple of 8.
    Has no gradient: an ``x`` that requires one is refused where it would be recorded.
    """
    logger.debug("GEMS PER TOKEN QUANT INT8")
    done = _cabi.host.token_quant_int8(x) if x.is_cuda else None
    if done is not None:
        return done
    assert x.dim() >= 1, "x needs a last dimension"
    if x.dtype not in _cabi.DTYPE_CODE:
        raise NotImplementedError(f"unsupported dtype {x.dtype}")
    _cabi.refuse_gradients(x=x)
    _cabi.require_cuda(x)
    k = x.shape[-1]
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    s = torch.empty(x.shape[:-1] + (1,), dtype=torch.float32, device=x.device)
    if k == 0:
        return q, s.fill_(1e-10 / 127.0)
    if x.numel() == 0:
        return q, s
    x2 = x.reshape(-1, k)
    if k > 1 and x2.stride(1) != 1:
        x2 = x2.contiguous()
    m = x2.shape[0]
    with _cabi.device_guard(x):
        _cabi.check(
            _cabi.lib().fg_per_token_quant_int8(
                _cabi.ptr(x2), _cabi.DTYPE_CODE[x.dtype], _cabi.ptr(q), _cabi.ptr(s), m, k,
                _cabi.row_stride(x2), k, None, 1, 0, None, _cabi.stream_ptr(x.device),
            )
        )
    return q, s
