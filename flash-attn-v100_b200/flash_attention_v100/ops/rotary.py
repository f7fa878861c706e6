"""Rotary positions: q and k turned by their positions before attention, with gradients.

The reference has none; its users rotate with elementwise torch operations, four passes over q and k and as many launches.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple, Union

import torch

from ..config import SUPPORTED_DTYPES
from ..kernels import _cabi
from ..kernels.tile_table import dtype_enum

_ROTARY_BYTES = ctypes.sizeof(_cabi.RotaryParams)


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: Optional[int] = None, turns_kept: float = 32.0, turns_stretched: float = 1.0,
                       device: Union[torch.device, str, None] = None) -> Tuple[torch.Tensor, float]:
    """(inv_freq, attention_factor): one frequency per pair of columns, in 64 bits, base ** (-2 i / rotary_dim), for
    rotary_embedding.  For contexts `factor` times as long as the model was trained for, `scaling` is

    "linear"    every frequency divided by factor (positions interpolated)
    "ntk"       a larger base, base * factor ** (d / (d - 2)): the highest frequency stays, the lowest is divided by factor
    "by_parts"  (Peng et al. 2023, YaRN) pairs that make turns_kept turns or more in original_length stay, those that make
                turns_stretched or fewer are divided by factor, a linear ramp between; attention_factor is 1 + ln(factor) / 10
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even, got {rotary_dim}")
    if not (base > 0 and factor > 0):
        raise ValueError("base and factor must be positive")
    half = rotary_dim // 2
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError('"ntk" needs a rotary_dim above 2')
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    elif scaling not in (None, "linear", "by_parts"):
        raise ValueError(f'scaling must be None, "linear", "ntk" or "by_parts", got {scaling!r}')
    freq = base ** (-torch.arange(half, dtype=torch.float64) / half)
    attention_factor = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "by_parts":
        if original_length is None or original_length <= 0:
            raise ValueError('"by_parts" needs original_length')
        if not turns_kept > turns_stretched:
            raise ValueError("turns_kept must be larger than turns_stretched")
        turns = original_length * freq / (2 * math.pi)
        kept = ((turns - turns_stretched) / (turns_kept - turns_stretched)).clamp(0.0, 1.0)
        freq = freq * kept + freq / factor * (1.0 - kept)
        attention_factor = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return (freq if device is None else freq.to(device)), attention_factor


def _operand(t: torch.Tensor) -> _cabi.Tensor4:
    return _cabi.Tensor4(t.data_ptr() or None, t.stride(0), t.stride(1), t.stride(2))


def _launch(xs, ys, positions, offset: int, inv_freq, interleaved: bool, factor: float, inverse: bool) -> None:
    x = xs[0]
    p = _cabi.RotaryParams()
    p.struct_bytes = _ROTARY_BYTES
    for i, (a, b) in enumerate(zip(xs, ys)):
        if a.numel():
            p.x[i], p.y[i], p.heads[i] = _operand(a), _operand(b), a.shape[2]
    if len(xs) == 2 and not xs[0].numel():              # the library's second tensor is the optional one
        p.x[0], p.y[0], p.heads[0] = p.x[1], p.y[1], p.heads[1]
        p.x[1], p.y[1], p.heads[1] = _cabi.Tensor4(), _cabi.Tensor4(), 0
    if positions is not None:
        p.positions = positions.data_ptr()
        p.positions_64bit = positions.dtype == torch.int64
        p.positions_stride_n = positions.stride(-1)
        p.positions_stride_b = positions.stride(0) if positions.dim() == 2 and positions.shape[0] > 1 else 0
    p.position0 = offset
    p.inv_freq = inv_freq.data_ptr()
    p.B, p.N, p.D, p.half = x.shape[0], x.shape[1], x.shape[3], inv_freq.shape[0]
    p.interleaved, p.inverse, p.factor = bool(interleaved), bool(inverse), factor
    p.dtype, p.device = dtype_enum(x.dtype), x.device.index
    p.stream = torch._C._cuda_getCurrentRawStream(x.device.index) or None
    _cabi.raise_for_status(_cabi.load().fa_b200_rotary(ctypes.byref(p)), "fa_b200_rotary")


def _unit_last(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(3) == 1 or t.numel() == 0 else t.contiguous()


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, positions, offset, inv_freq, interleaved, factor, inverse, *xs):
        xs = [_unit_last(x) for x in xs]
        ys = tuple(torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in xs)
        _launch(xs, ys, positions, offset, inv_freq, interleaved, factor, inverse)
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = (offset, interleaved, factor, inverse)
        ctx.set_materialize_grads(False)
        return ys

    @staticmethod
    def backward(ctx, *grads):
        # the gradient of a turn is the turn back, which has a gradient of its own
        positions, inv_freq = ctx.saved_tensors
        offset, interleaved, factor, inverse = ctx.how
        wanted = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[6 + i]]
        out = [None] * len(grads)
        if wanted:
            for i, d in zip(wanted, _Rotary.apply(positions, offset, inv_freq, interleaved, factor, not inverse, *(grads[i] for i in wanted))):
                out[i] = d
        return (None,) * 6 + tuple(out)


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor] = None, *, inv_freq: torch.Tensor,
                     positions: Union[torch.Tensor, int, None] = None, interleaved: bool = False, attention_factor: float = 1.0,
                     inplace: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """q, or (q, k), turned by position; one launch, and one for the gradients of both, which have gradients of their own.

    The columns of a head are taken in pairs (u, w), the i-th of angle a = position * inv_freq[i]:
        u' = attention_factor (u cos a - w sin a),  w' = attention_factor (w cos a + u sin a)

    Args:
        q, k: [batch, seq_len, heads, head_dim] fp16, bf16 or fp32, head_dim up to 128; k may have its own number of heads
        inv_freq: (pairs,) frequencies on the same device (rotary_frequencies; used in 64 bits); columns from 2 * pairs on
            stay as they are
        positions: of the tokens, int32 or int64 (seq_len,), (1, seq_len) or (batch, seq_len), e.g. KeyRanges.positions; an int:
            that of the first token (default 0), the others follow
        interleaved: pairs are neighbouring columns 2i, 2i + 1 instead of i, i + pairs
        inplace: write over q and k (no gradients), e.g. rows of a key cache
    """
    if not inplace and type(attention_factor) is float and not torch.compiler.is_compiling():
        result = _cabi.load_op().rotary(q, k, positions, inv_freq, bool(interleaved), attention_factor)
        if result is not None:
            return result
    xs = (q,) if k is None else (q, k)
    for name, x in zip("qk", xs):
        if not isinstance(x, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if x.dim() != 4:
            raise ValueError("Input tensors must be 4-dimensional [batch, seq_len, num_heads, head_dim]")
        if x.device.type != "cuda":
            raise ValueError("rotary_embedding requires CUDA tensors")
        if x.dtype not in SUPPORTED_DTYPES:
            raise ValueError(f"Unsupported dtype {x.dtype}. Supported types: {', '.join(str(d) for d in SUPPORTED_DTYPES)}")
        if x.dtype != q.dtype or x.device != q.device or (x.shape[0], x.shape[1], x.shape[3]) != (q.shape[0], q.shape[1], q.shape[3]):
            raise ValueError("q and k must match in batch, seq_len, head_dim, dtype and device")
    B, N, _, D = q.shape
    if D > 128:
        raise ValueError(f"head_dim {D} is not supported (maximum 128)")
    if not isinstance(inv_freq, torch.Tensor):
        raise TypeError("inv_freq must be a torch.Tensor")
    if inv_freq.dim() != 1 or not inv_freq.is_floating_point() or 2 * inv_freq.shape[0] > D:
        raise ValueError(f"inv_freq must be a 1-dimensional floating-point tensor of at most head_dim / 2 = {D // 2} values")
    if inv_freq.device != q.device:
        raise ValueError("inv_freq must be on the same device as q")
    if inv_freq.requires_grad:
        raise ValueError("inv_freq has no gradient here: detach it")
    if inv_freq.dtype != torch.float64 or not inv_freq.is_contiguous():
        inv_freq = inv_freq.to(torch.float64).contiguous()
    offset = 0
    if isinstance(positions, torch.Tensor):
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
        if positions.device != q.device:
            raise ValueError("positions must be on the same device as q")
        if tuple(positions.shape) not in ((N,), (1, N), (B, N)):
            raise ValueError(f"positions have shape {tuple(positions.shape)}, expected ({N},), (1, {N}) or ({B}, {N})")
    elif positions is not None:
        offset = int(positions)
        if offset != positions or not -2 ** 63 <= offset < 2 ** 63:
            raise ValueError(f"positions must be a tensor or a whole number of 64 bits, got {positions!r}")
        positions = None
    wants = torch.is_grad_enabled() and any(x.requires_grad for x in xs)
    if inplace:
        if wants:
            raise ValueError("inplace=True is for calls without gradients")
        for x in xs:
            if x.numel() and (x.stride(3) != 1 or any(s == 0 and n > 1 for s, n in zip(x.stride(), x.shape))):
                raise ValueError("inplace=True needs tensors with a contiguous head dimension and rows of their own")
        if k is not None and q.numel() and k.numel() and q.data_ptr() == k.data_ptr():
            raise ValueError("inplace=True needs q and k that do not share memory")
        ys = xs
        if not all(x.numel() == 0 for x in xs):
            _launch(xs, ys, positions, offset, inv_freq, interleaved, float(attention_factor), False)
        torch.autograd.graph.increment_version(list(xs))
    elif wants:
        ys = _Rotary.apply(positions, offset, inv_freq, interleaved, float(attention_factor), False, *xs)
    else:
        ins = [_unit_last(x) for x in xs]
        ys = tuple(torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in xs)
        if not all(x.numel() == 0 for x in xs):
            _launch(ins, ys, positions, offset, inv_freq, interleaved, float(attention_factor), False)
    return ys[0] if k is None else (ys[0], ys[1])


__all__ = ["rotary_embedding", "rotary_frequencies"]
