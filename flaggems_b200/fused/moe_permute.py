"""moe_permute / moe_unpermute: tokens sorted by expert and back, with router weights, and their gradients.

    rows, row_scale, plan = moe_permute(hidden_states, topk_ids, num_experts)
    ...                                    # the experts, e.g. w8a8_int8_grouped_mm with plan.offs
    out = moe_unpermute(rows, plan, topk_weights)

The reference has no such pair: its expert kernel gathers tokens by ``sorted_token_ids`` and ``moe_sum`` adds rows in
slot order (src/flag_gems/fused/fused_moe.py:1101-1110, src/flag_gems/fused/moe_sum.py:24-67), which serves its own layer
and has no backward pass.  These serve experts that run outside ``fused_experts_impl``, in training too.
"""
import logging
from typing import NamedTuple, Optional, Tuple

import torch

from .. import _cabi

logger = logging.getLogger(__name__.replace("flaggems_b200", "flag_gems", 1))

_ELEMENT_BYTES = {torch.bfloat16: 2, torch.float16: 2, torch.float32: 4, torch.int8: 1, torch.uint8: 1,
                  torch.float8_e4m3fn: 1, torch.float8_e5m2: 1}


class MoEPermutation(NamedTuple):
    """Where ``moe_permute`` put the tokens; ``moe_unpermute`` takes it as it is."""

    offs: torch.Tensor  #: int32 [num_experts]: rows [offs[e - 1], offs[e]) are expert e's
    row_of_slot: torch.Tensor  #: int32 [tokens, topk]: the slot's row, ~row (negative) without an expert
    slot_of_row: torch.Tensor  #: int32 [tokens * topk]: token * topk + k; ascending within an expert


def _rows(t, what):
    """2-D rows with contiguous values (copied only where they are not)."""
    assert t.dim() == 2, f"{what} must be 2-D"
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _check_devices(first, *others):
    _cabi.require_cuda(first, *others)
    for t in others:
        assert t is None or t.device == first.device, f"operands on {first.device} and {t.device}"


def _refuse_tangents(*tensors):
    if any(t is not None and _cabi.has_tangent(t) for t in tensors):
        raise NotImplementedError("moe_permute and moe_unpermute have no forward-mode derivative")


def _permute(x, topk_ids, num_experts, scale, expert_map):
    tokens, topk = topk_ids.shape
    hidden = x.shape[1]
    n = tokens * topk
    dev = x.device
    rows = torch.empty((n, hidden), dtype=x.dtype, device=dev)
    row_scale = None if scale is None else torch.empty((n, scale.shape[1]), dtype=torch.float32, device=dev)
    offs = torch.empty(num_experts, dtype=torch.int32, device=dev)
    row_of_slot = torch.empty((tokens, topk), dtype=torch.int32, device=dev)
    slot_of_row = torch.empty(n, dtype=torch.int32, device=dev)
    with _cabi.device_guard(x):
        need = max(int(_cabi.lib().fg_moe_permute_workspace_bytes(tokens, topk, num_experts)), 0)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        _cabi.check(_cabi.lib().fg_moe_permute(
            _cabi.ptr(rows), _cabi.ptr(row_scale), _cabi.ptr(offs), _cabi.ptr(row_of_slot), _cabi.ptr(slot_of_row),
            _cabi.ptr(x), _cabi.ptr(scale), _cabi.ptr(topk_ids), 1 if topk_ids.dtype == torch.int64 else 0,
            _cabi.ptr(expert_map), 0 if expert_map is None else expert_map.numel(), tokens, topk, num_experts, hidden,
            _ELEMENT_BYTES[x.dtype], x.stride(0), 0 if scale is None else scale.shape[1],
            0 if scale is None else scale.stride(0), _cabi.ptr(ws), need, _cabi.stream_ptr(dev)))
    return rows, row_scale, offs, row_of_slot, slot_of_row


def _unpermute(rows, row_of_slot, weights):
    tokens, topk = row_of_slot.shape
    out = torch.empty((tokens, rows.shape[1]), dtype=rows.dtype, device=rows.device)
    with _cabi.device_guard(rows):
        _cabi.check(_cabi.lib().fg_moe_unpermute(
            _cabi.ptr(out), _cabi.ptr(rows), _cabi.ptr(row_of_slot), _cabi.ptr(weights),
            0 if weights is None else _cabi.DTYPE_CODE[weights.dtype], tokens, topk, rows.shape[0], rows.shape[1],
            rows.stride(0), 0 if weights is None else weights.stride(0), _cabi.DTYPE_CODE[rows.dtype],
            _cabi.stream_ptr(rows.device)))
    return out


class _Permute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, topk_ids, num_experts, scale, expert_map):
        rows, row_scale, offs, row_of_slot, slot_of_row = _permute(x, topk_ids, num_experts, scale, expert_map)
        ctx.save_for_backward(row_of_slot)
        ctx.mark_non_differentiable(*(t for t in (row_scale, offs, row_of_slot, slot_of_row) if t is not None))
        return rows, row_scale, offs, row_of_slot, slot_of_row

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_rows, *_):
        _refuse_tangents(d_rows)
        row_of_slot, = ctx.saved_tensors
        return _unpermute(_rows(d_rows, "the gradient"), row_of_slot, None), None, None, None, None


class _Unpermute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, row_of_slot, weights):
        ctx.save_for_backward(rows if ctx.needs_input_grad[2] else None, row_of_slot, weights)
        ctx.rows_shape = rows.shape
        return _unpermute(rows, row_of_slot, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        _refuse_tangents(d_out)
        rows, row_of_slot, weights = ctx.saved_tensors
        d_out = _rows(d_out, "the gradient")
        d_rows = d_weights = None
        if ctx.needs_input_grad[0]:
            d_rows = torch.empty(ctx.rows_shape, dtype=d_out.dtype, device=d_out.device)
        if ctx.needs_input_grad[2]:
            d_weights = torch.empty(weights.shape, dtype=weights.dtype, device=weights.device)
        tokens, topk = row_of_slot.shape
        with _cabi.device_guard(d_out):
            _cabi.check(_cabi.lib().fg_moe_unpermute_backward(
                _cabi.ptr(d_rows), _cabi.ptr(d_weights), _cabi.ptr(d_out), _cabi.ptr(rows), _cabi.ptr(row_of_slot),
                _cabi.ptr(weights), 0 if weights is None else _cabi.DTYPE_CODE[weights.dtype], tokens, topk,
                ctx.rows_shape[0], ctx.rows_shape[1], d_out.stride(0), 0 if rows is None else rows.stride(0),
                0 if weights is None else weights.stride(0), _cabi.DTYPE_CODE[d_out.dtype],
                _cabi.stream_ptr(d_out.device)))
        return d_rows, None, d_weights


def moe_permute(
    hidden_states: torch.Tensor,
    topk_ids: torch.Tensor,
    num_experts: int,
    scale: Optional[torch.Tensor] = None,
    expert_map: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor], MoEPermutation]:
    """Copies every token's row to one row per route slot, sorted by expert (ascending slots within an expert).

    ``hidden_states`` [tokens, hidden] in bf16, fp16, fp32, int8, uint8 or an 8-bit float; ``topk_ids`` int32 or int64
    [tokens, topk]; at most 1024 experts.  ``scale`` float32 [tokens, any]: the scales of quantised rows, carried along.
    ``expert_map`` int32 or int64: the expert of an id, for ranks that hold some of the experts; ``num_experts`` counts
    those.  Slots whose id (or mapped id) is outside [0, num_experts) have no expert: their rows follow offs[-1], are
    zeros (their scales ones) and get no gradient back.

    Returns ``(rows [tokens * topk, hidden], row_scale or None, plan)``; ``plan.offs`` is what
    ``w8a8_int8_grouped_mm`` and ``scaled_grouped_mm`` take.  Differentiable in ``hidden_states`` of
    bf16, fp16 and fp32, once and in reverse mode.  A step that is captured into a CUDA graph with its backward pass takes
    leaves of its own, as with every operator of torch.
    """
    logger.debug("GEMS MOE PERMUTE")
    if hidden_states.is_cuda:
        done = _cabi.host.moe_permute(hidden_states, topk_ids, num_experts, scale, expert_map)
        if done is not None:
            return done[0], done[1], MoEPermutation(*done[2:])
    assert topk_ids.dim() == 2, "topk_ids must be [tokens, topk]"
    if topk_ids.dtype not in (torch.int32, torch.int64):
        raise NotImplementedError(f"topk_ids must be int32 or int64, got {topk_ids.dtype}")
    if hidden_states.dtype not in _ELEMENT_BYTES:
        raise NotImplementedError(f"unsupported dtype {hidden_states.dtype}")
    if hidden_states.dtype not in _cabi.DTYPE_CODE and hidden_states.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"hidden_states of {hidden_states.dtype} have no gradient")
    num_experts = int(num_experts)
    assert num_experts > 0, "num_experts must be positive"
    x = _rows(hidden_states, "hidden_states")
    assert x.shape[0] == topk_ids.shape[0], f"{x.shape[0]} tokens, {topk_ids.shape[0]} rows of topk_ids"
    if scale is not None:
        assert scale.dtype == torch.float32, "scale must be float32"
        scale = _rows(scale, "scale")
        assert scale.shape[0] == x.shape[0], f"{x.shape[0]} tokens, {scale.shape[0]} rows of scales"
        if scale.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("scale has no gradient")
    _refuse_tangents(x, scale)
    if expert_map is not None:
        assert expert_map.dim() == 1 and expert_map.numel() > 0, "expert_map must be 1-D and not empty"
        if expert_map.dtype not in (torch.int32, torch.int64):
            raise NotImplementedError(f"expert_map must be int32 or int64, got {expert_map.dtype}")
    _check_devices(x, topk_ids, scale, expert_map)
    topk_ids = topk_ids.contiguous()
    if expert_map is not None:
        if expert_map.dtype == torch.int64:  # what is outside the range stays outside in 32 bits
            expert_map = expert_map.clamp(-1, num_experts).to(torch.int32)
        expert_map = expert_map.contiguous()
    call = _Permute.apply if torch.is_grad_enabled() and x.requires_grad else _permute
    rows, row_scale, *plan = call(x, topk_ids, num_experts, scale, expert_map)
    return rows, row_scale, MoEPermutation(*plan)


def moe_unpermute(
    rows: torch.Tensor,
    plan: MoEPermutation,
    topk_weights: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``out[t] = sum_k topk_weights[t, k] * rows[plan.row_of_slot[t, k]]``, summed in fp32 in slot order.

    ``rows`` [tokens * topk, hidden] in bf16, fp16 or fp32; ``plan`` from ``moe_permute``; ``topk_weights``
    [tokens, topk] in bf16, fp16 or fp32, None for ones.  Slots without an expert add nothing and their rows are not
    read.  Returns [tokens, hidden] of the type of ``rows``.  Differentiable in ``rows`` and ``topk_weights``, once and in
    reverse mode.
    """
    logger.debug("GEMS MOE UNPERMUTE")
    if rows.is_cuda:
        out = _cabi.host.moe_unpermute(rows, plan.row_of_slot, topk_weights)
        if out is not None:
            return out
    if rows.dtype not in _cabi.DTYPE_CODE:
        raise NotImplementedError(f"unsupported dtype {rows.dtype}")
    row_of_slot = plan.row_of_slot
    assert row_of_slot.dim() == 2 and row_of_slot.dtype == torch.int32, "plan.row_of_slot must be int32 [tokens, topk]"
    rows = _rows(rows, "rows")
    assert rows.shape[0] == row_of_slot.numel(), f"the plan has {row_of_slot.numel()} rows, got {rows.shape[0]}"
    if topk_weights is not None:
        assert topk_weights.shape == row_of_slot.shape, f"topk_weights must have shape {tuple(row_of_slot.shape)}"
        if topk_weights.dtype not in _cabi.DTYPE_CODE:
            raise NotImplementedError(f"unsupported dtype of topk_weights {topk_weights.dtype}")
        topk_weights = _rows(topk_weights, "topk_weights")
    _refuse_tangents(rows, topk_weights)
    _check_devices(rows, row_of_slot, topk_weights)
    row_of_slot = row_of_slot.contiguous()
    if torch.is_grad_enabled() and (rows.requires_grad or (topk_weights is not None and topk_weights.requires_grad)):
        return _Unpermute.apply(rows, row_of_slot, topk_weights)
    return _unpermute(rows, row_of_slot, topk_weights)
