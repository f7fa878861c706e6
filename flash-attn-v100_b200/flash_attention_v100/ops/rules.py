"""Attention whose scores are capped, moved by the distance between query and key, or limited to a range of keys a row:

    x = cap tanh(scale q.k / cap) - slope_h |position - key|,  softmax over the row's range

The autograd op behind flash_attention_v100_with_rules.  The reference has no such form.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from ..kernels import _cabi
from .attention import _base_params, _tensor4, _variant_override
from ..utils import _last_dim_contiguous, last_derivative
from .key_ranges import KeyRanges, check_plan

_RULES_BYTES = ctypes.sizeof(_cabi.RuleParams)


def _rules(cap: float, slopes: Optional[torch.Tensor], plan: torch.Tensor, plan_batch: int, max_keys: int = 0) -> _cabi.RuleParams:
    return _cabi.RuleParams(_RULES_BYTES, plan.data_ptr(), plan_batch, cap, slopes.data_ptr() if slopes is not None else None, max_keys)


def check_rules(q: torch.Tensor, k: torch.Tensor, score_cap: Optional[float], slopes: Optional[torch.Tensor],
                ranges: Optional[KeyRanges]) -> Tuple[float, Optional[torch.Tensor]]:
    """(cap or 0, slopes ready for the kernels); raises what the public entry raises."""
    cap = 0.0
    if score_cap is not None:
        cap = float(score_cap)
        if not 0.0 < cap < 1e30 or ctypes.c_float(cap).value == 0.0:        # (a 0 would mean none to the kernels)
            raise ValueError(f"score_cap must be positive and finite in 32 bits, got {score_cap}")
    if slopes is not None:
        if not isinstance(slopes, torch.Tensor):
            raise TypeError("distance_slopes must be a torch.Tensor")
        if tuple(slopes.shape) != (q.shape[2],) or not slopes.is_floating_point():
            raise ValueError(f"distance_slopes must be a floating-point tensor of shape ({q.shape[2]},), got {tuple(slopes.shape)}")
        if slopes.device != q.device:
            raise ValueError("distance_slopes must be on the same device as input tensors")
        if slopes.requires_grad:
            raise ValueError("distance_slopes have no gradient here: detach them")
        if slopes.dtype != torch.float32 or not slopes.is_contiguous():
            slopes = slopes.to(torch.float32).contiguous()
    if ranges is not None:
        if not isinstance(ranges, KeyRanges):
            raise TypeError("key_ranges must be a KeyRanges (build_key_ranges)")
        if (ranges.seq_q, ranges.seq_k) != (q.shape[1], k.shape[1]) or ranges.batch not in (1, q.shape[0]):
            raise ValueError(f"key_ranges are for batch {ranges.batch}, {ranges.seq_q} rows and {ranges.seq_k} keys; "
                             f"the call has batch {q.shape[0]}, {q.shape[1]} rows and {k.shape[1]} keys")
        if ranges.device != q.device:
            raise ValueError("key_ranges must be on the same device as input tensors")
        check_plan(ranges)
    return cap, slopes


def native_call_rules(q, k, v, scale, score_cap, slopes, ranges: KeyRanges):
    """(o, lse) by the native operator, or None where it does not serve the call (as attention.native_call)."""
    if torch.compiler.is_compiling() or getattr(_variant_override, "value", _cabi.VARIANT_AUTO) != _cabi.VARIANT_AUTO:
        return None
    return _cabi.load_op().attention_rules(q, k, v, scale, score_cap, slopes, ranges.plan, ranges.batch, ranges.seq_q, ranges.seq_k, ranges.max_keys)


def launch_forward_rules(q, k, v, scale, cap, slopes, plan, plan_batch, o_residual=None, split_keys=False, max_keys=0):
    """(o, lse) <- fa_b200_fwd_with_rules; arguments as launch_forward's."""
    B, Nq, H, _ = q.shape
    o = q.new_empty(q.shape)
    lse = q.new_empty((B, H, Nq), dtype=torch.float32)
    if k.shape[1] == 0:                                   # no keys at all: every row sees nothing
        if o_residual is not None:
            o_residual.zero_()
        return o.zero_(), lse.fill_(float("-inf"))
    p = _base_params(q, k, v, o, lse, scale, False, 0.0, 0, 0)
    if o_residual is not None:
        p.o_lo = _tensor4(o_residual)
    lib = _cabi.load()
    r = _rules(cap, slopes, plan, plan_batch, max_keys)
    nbytes = int(lib.fa_b200_fwd_rules_workspace_bytes(ctypes.byref(p), ctypes.byref(r))) if split_keys else 0
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    rc = lib.fa_b200_fwd_with_rules(ctypes.byref(p), ctypes.byref(r), ws.data_ptr() if nbytes else None, nbytes)
    _cabi.raise_for_status(rc, "fa_b200_fwd_with_rules")
    return o, lse


def launch_backward_rules(d_o, q, k, v, o, lse, scale, cap, slopes, plan, plan_batch, o_residual=None):
    """(dq, dk, dv) <- fa_b200_bwd_with_rules."""
    if k.shape[1] == 0:
        return torch.zeros_like(q), torch.empty_like(k), torch.empty_like(v)
    d_o = _last_dim_contiguous(d_o)
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    p = _base_params(q, k, v, o, lse, scale, False, 0.0, 0, 0, d_o=d_o, dq=dq, dk=dk, dv=dv)
    if o_residual is not None:
        p.o_lo = _tensor4(o_residual)
    lib = _cabi.load()
    nbytes = int(lib.fa_b200_bwd_rules_workspace_bytes(ctypes.byref(p)))
    ws = q.new_empty(nbytes, dtype=torch.uint8)
    p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
    r = _rules(cap, slopes, plan, plan_batch)
    _cabi.raise_for_status(lib.fa_b200_bwd_with_rules(ctypes.byref(p), ctypes.byref(r)), "fa_b200_bwd_with_rules")
    return dq, dk, dv


class RuledAttentionFunction(torch.autograd.Function):
    """(o, lse) of q, k, v under rules; the lse is not differentiable."""

    @staticmethod
    def forward(ctx, q, k, v, scale, cap, slopes, plan, plan_batch, max_keys):
        # what rounding o to 16 bits dropped goes to the backward: without it half of the error of fp16 dQ and dK was delta's
        needs_grad = any(ctx.needs_input_grad[:3])
        o_lo = torch.empty(q.shape, dtype=q.dtype, device=q.device) if needs_grad and q.dtype != torch.float32 else None
        o, lse = launch_forward_rules(q, k, v, scale, cap, slopes, plan, plan_batch, o_residual=o_lo, split_keys=not needs_grad, max_keys=max_keys)
        ctx.save_for_backward(q, k, v, o, lse, slopes, plan, o_lo)
        ctx.how = (scale, cap, plan_batch)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @last_derivative
    def backward(ctx, grad_o, _grad_lse=None):
        q, k, v, o, lse, slopes, plan, o_lo = ctx.saved_tensors
        scale, cap, plan_batch = ctx.how
        if grad_o is None:
            return (None,) * 9
        grads = launch_backward_rules(grad_o, q, k, v, o, lse, scale, cap, slopes, plan, plan_batch, o_residual=o_lo)
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None,) * 6


__all__ = ["RuledAttentionFunction", "check_rules", "launch_forward_rules", "launch_backward_rules"]
