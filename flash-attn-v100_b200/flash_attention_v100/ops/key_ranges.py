"""Key ranges: which keys each query sees, as one interval [first, end) a row.

Packed documents, visible prefixes, sliding windows, causal masks and caches of ragged lengths are all such intervals.
They are built on the GPU from lengths, once a step, and read by the attention of every layer
(`flash_attention_v100_with_rules(..., key_ranges=)`); whole key blocks that no row of a query tile sees are skipped.
The reference expands masks to a dense bias instead (examples/basic_usage.py:228-250).
"""
from __future__ import annotations

import ctypes
import operator
from typing import Optional, Union

import torch

from ..kernels import _cabi

_INT32_MAX = 2 ** 31 - 1
_RANGES_BYTES = ctypes.sizeof(_cabi.RangesParams)


def _ceil128(n: int) -> int:
    return -(-n // 128) * 128


class KeyRanges:
    """The keys each query row sees, and what the kernels want to know of 128 rows at once.  Made by build_key_ranges.

    first, end: (batch, seq_q) int32, row i of entry b sees keys [first, end) (0, 0: none)
    positions:  (batch, seq_q) int32, the row's place within its document, for rotary_embedding
    """
    __slots__ = ("plan", "positions", "batch", "seq_q", "seq_k", "max_keys", "_first", "_end")

    def __init__(self, plan: torch.Tensor, positions: torch.Tensor, batch: int, seq_q: int, seq_k: int, max_keys: int = 0,
                 first: Optional[torch.Tensor] = None, end: Optional[torch.Tensor] = None):
        self.plan, self.positions = plan, positions
        self.batch, self.seq_q, self.seq_k = batch, seq_q, seq_k
        self.max_keys = max_keys                # most keys a row sees (0: not known), for how the work is divided
        self._first, self._end = first, end

    @property
    def device(self) -> torch.device:
        return self.plan.device

    def _column(self, at: int) -> torch.Tensor:
        return self.plan.as_strided((self.batch, self.seq_q), (2 * _ceil128(self.seq_q), 2), at if self.batch and self.seq_q else 0)

    @property
    def first(self) -> torch.Tensor:
        return self._column(0) if self._first is None else self._first

    @property
    def end(self) -> torch.Tensor:
        return self._column(1) if self._end is None else self._end


def check_plan(r: KeyRanges) -> None:
    """Raises where r cannot be what build_key_ranges made: the kernels read, and a build writes, as many bytes as its sizes say."""
    need = _cabi.load().fa_b200_key_ranges_bytes(r.batch, r.seq_q, r.seq_k) // 4
    if r.plan.dtype != torch.int32 or not r.plan.is_contiguous() or r.plan.numel() < need:
        raise ValueError(f"a plan for batch {r.batch}, {r.seq_q} rows and {r.seq_k} keys is {need} dense int32, got "
                         f"{r.plan.numel()} of {r.plan.dtype}: KeyRanges come from build_key_ranges")


def _lengths(name: str, t: Optional[torch.Tensor], shapes, device: torch.device) -> Optional[torch.Tensor]:
    """Whole numbers on the device as dense int32."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int32 or int64, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    if tuple(t.shape) not in shapes:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected one of {shapes}")
    t = t.detach()
    if t.dtype != torch.int32:
        t = t.clamp(-_INT32_MAX, _INT32_MAX).to(torch.int32)         # (a length beyond 32 bits means all there is)
    return t if t.is_contiguous() else t.contiguous()


def _start(query_offsets) -> int:
    """query_offsets where it is no tensor."""
    if query_offsets is None:
        return 0
    try:
        start = operator.index(query_offsets)
    except TypeError:
        raise TypeError(f"query_offsets must be a tensor or a whole number, got {type(query_offsets).__name__}") from None
    if not -_INT32_MAX - 1 <= start <= _INT32_MAX:
        raise ValueError(f"query_offsets {start} does not fit 32 bits")
    return start


def _most(causal: bool, window: Optional[int]) -> int:
    return 0 if window is None else min(window if causal else 2 * window - 1, _INT32_MAX)


def _device_index(device, *tensors) -> Optional[int]:
    """The CUDA device the ranges are built on, None where there is no GPU or it is another kind of device."""
    if device is None:
        device = next((t.device for t in tensors if isinstance(t, torch.Tensor)), None)
        if device is None:
            return torch.cuda.current_device() if torch.cuda.is_available() else None
    elif not isinstance(device, torch.device):
        device = torch.device(device)
    if device.type != "cuda" or not torch.cuda.is_available():
        return None
    return torch.cuda.current_device() if device.index is None else device.index


def build_key_ranges(seq_q: int, seq_k: int, *, batch: int = 1, causal: bool = False, window: Optional[int] = None,
                     document_offsets: Optional[torch.Tensor] = None, prefix_lengths: Optional[torch.Tensor] = None,
                     key_lengths: Optional[torch.Tensor] = None, query_offsets: Union[torch.Tensor, int, None] = None,
                     rows: Optional[torch.Tensor] = None, device: Union[torch.device, str, int, None] = None,
                     out: Optional[KeyRanges] = None) -> KeyRanges:
    """Build a KeyRanges on the GPU.

    Row i of batch entry b stands at position t = i + query_offsets[b] (an int: of every entry; default 0).  Without documents
    rows at t < 0 (more queries than a cache has keys) go by the same rules: under causal they see no key but a prefix, else the
    keys of their window, or all.

    Args:
        seq_q, seq_k: rows and keys of the attention calls;  batch: entries, 1 serves any batch
        causal: keys up to the row's own position
        window: keys at most window - 1 back (and, without causal, ahead)
        document_offsets: (batch, documents + 1) or (documents + 1,) ascending boundaries; a row sees keys of its own
            document only, rows before the first and behind the last boundary see nothing
        prefix_lengths: causal without a window only: the first keys of a document that all of its rows see; (batch, documents)
            or (documents,), without documents (batch,)
        key_lengths: (batch,) keys there are; 0 hides all
        query_offsets: (batch,) tensor, for queries at the end of a cache: key_lengths - seq_q
        rows: (batch, seq_q, 2) intervals given by hand instead of all of the above but query_offsets
        device: of the plan; default that of the first tensor, else the current one
        out: an earlier KeyRanges of the same sizes, written anew in place (a captured graph reads it again).  A backward
            whose forward read its earlier contents raises
    """
    offset_tensor = query_offsets if isinstance(query_offsets, torch.Tensor) else None
    start = 0 if offset_tensor is not None else _start(query_offsets)
    if out is None and rows is None and (window is None or window >= 1) and not torch.compiler.is_compiling():
        # (None: a form the native operator does not serve, or one that is refused below)
        index = _device_index(device, document_offsets, prefix_lengths, key_lengths, offset_tensor)
        if index is not None:
            result = _cabi.load_op().key_ranges(seq_q, seq_k, batch, bool(causal), window or 0, document_offsets, prefix_lengths, key_lengths, offset_tensor, start, index)
            if result is not None:
                return KeyRanges(result[0], result[1], batch, seq_q, seq_k, _most(causal, window), result[2], result[3])
    if seq_q < 0 or seq_k < 0 or batch < 0:
        raise ValueError(f"sizes must not be negative (seq_q {seq_q}, seq_k {seq_k}, batch {batch})")
    if max(seq_q, seq_k, batch) > _INT32_MAX:
        raise ValueError(f"sizes must be below 2**31 (seq_q {seq_q}, seq_k {seq_k}, batch {batch})")
    if window is not None and not 1 <= window <= _INT32_MAX:
        raise ValueError(f"window must be at least 1, got {window}")
    if prefix_lengths is not None and (not causal or window is not None):
        raise ValueError("prefix_lengths are defined for causal ranges without a window")
    if rows is not None and (causal or window is not None or document_offsets is not None or key_lengths is not None):
        raise ValueError("rows are the ranges: causal, window, document_offsets, prefix_lengths and key_lengths cannot be combined with them")
    if device is None:
        given = next((t for t in (document_offsets, prefix_lengths, key_lengths, offset_tensor, rows) if t is not None), None)
        device = given.device if given is not None else (out.device if out is not None else torch.device("cuda"))
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError(f"key ranges are built on a CUDA device, got {device}")
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    documents = 0
    if document_offsets is not None:
        documents = document_offsets.shape[-1] - 1 if document_offsets.dim() else 0
        if documents < 1:
            raise ValueError("document_offsets need two boundaries or more")
    offsets = _lengths("document_offsets", document_offsets, [(batch, documents + 1), (documents + 1,)], device)
    prefixes = _lengths("prefix_lengths", prefix_lengths, [(batch, documents), (documents,)] if documents else [(batch,)], device)
    lengths = _lengths("key_lengths", key_lengths, [(batch,)], device)
    starts = _lengths("query_offsets", offset_tensor, [(batch,)], device)
    given = _lengths("rows", rows, [(batch, seq_q, 2)], device)
    lib = _cabi.load()
    nbytes = lib.fa_b200_key_ranges_bytes(batch, seq_q, seq_k)
    if out is None:
        out = KeyRanges(torch.empty(nbytes // 4, dtype=torch.int32, device=device),
                        torch.empty((batch, seq_q), dtype=torch.int32, device=device), batch, seq_q, seq_k, _most(causal, window))
    else:
        if (out.batch, out.seq_q, out.seq_k) != (batch, seq_q, seq_k) or out.device != device:
            raise ValueError(f"out is for batch {out.batch}, {out.seq_q} rows and {out.seq_k} keys on {out.device}")
        check_plan(out)
        if tuple(out.positions.shape) != (batch, seq_q) or out.positions.dtype != torch.int32 or not out.positions.is_contiguous() or \
                out.positions.device != device:
            raise ValueError("out.positions are not build_key_ranges'")
        torch.autograd.graph.increment_version([out.plan, out.positions])
        out.max_keys = _most(causal, window)
    p = _cabi.RangesParams(
        _RANGES_BYTES, out.plan.data_ptr(), nbytes, out.positions.data_ptr(), given.data_ptr() if given is not None else None,
        offsets.data_ptr() if offsets is not None else None, prefixes.data_ptr() if prefixes is not None else None,
        lengths.data_ptr() if lengths is not None else None, starts.data_ptr() if starts is not None else None,
        documents + 1 if offsets is not None and offsets.dim() == 2 else 0,
        (documents if prefixes.dim() == 2 else (0 if documents else 1)) if prefixes is not None else 0,
        documents, start, bool(causal), window or 0,
        batch, seq_q, seq_k, device.index, torch._C._cuda_getCurrentRawStream(device.index) or None)
    _cabi.raise_for_status(lib.fa_b200_key_ranges(ctypes.byref(p)), "fa_b200_key_ranges")
    return out


__all__ = ["KeyRanges", "build_key_ranges"]
