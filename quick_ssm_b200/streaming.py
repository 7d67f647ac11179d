"""Stateful forward scan: feed a sequence in pieces and carry the hidden state between calls.

The recurrence needs nothing from the past except ``h`` at the last step, so inference over a
stream (or token-by-token decoding) is a chain of ordinary forward scans, each seeded with the
state the previous one left (``h_in`` / ``h_last`` of the C ABI).  The reference lists a fast
inference mode as future work; its block scan has no way to pass a state in.

``gated_scan_chunk`` is the same for the scan with the layer's gate activations fused in
(``gated.gated_scan``): the form a serving layer calls for prompts and for single tokens.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .gated import _fusable, _gates
from .scan_interface import _kernel_out_dtype, _prepare_inputs


class ScanState:
    """Hidden state ``h`` after the last step seen, ``[B, D]`` fp32 on the device."""

    def __init__(self, h: torch.Tensor):
        if h.dim() != 2 or h.dtype != torch.float32:
            raise ValueError("state must be a [B, D] float32 tensor")
        self.h = h

    @classmethod
    def zeros(cls, batch: int, channels: int, device="cuda") -> "ScanState":
        return cls(torch.zeros((batch, channels), dtype=torch.float32, device=device))

    def clone(self) -> "ScanState":
        return ScanState(self.h.clone())


@torch.no_grad()
def scan_chunk(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, c: Optional[torch.Tensor],
               state: Optional[ScanState] = None, *, out_dtype: Optional[torch.dtype] = None
               ) -> Tuple[torch.Tensor, ScanState]:
    """Forward scan over one piece ``[B, L_piece, D]`` of a longer sequence.

    Returns ``(y, new_state)`` with ``y = c*h`` (or ``h`` itself when ``c`` is None).  Passing the
    returned state to the next call continues the same recurrence; the concatenated outputs equal
    one scan over the concatenated inputs up to fp32 rounding of the carried state.
    """
    if x.dim() != 3 or x.shape != a.shape or x.shape != b.shape or (c is not None and c.shape != x.shape):
        raise ValueError("x, a, b, c must share the same shape [B, L, D].")
    B, L, D = x.shape
    if state is not None and tuple(state.h.shape) != (B, D):
        raise ValueError(f"state is {tuple(state.h.shape)}, expected {(B, D)}")
    xs, as_, bs, cs = _prepare_inputs(x, a, b, c)
    out_dtype = out_dtype or x.dtype
    k_out = _kernel_out_dtype(xs.dtype, out_dtype)
    y = torch.empty((B, L, D), dtype=k_out, device=x.device)
    h_last = torch.empty((B, D), dtype=torch.float32, device=x.device)
    _lib.scan_fwd(xs, as_, bs, cs, y, h_in=None if state is None else state.h.contiguous(), h_last=h_last)
    return (y if k_out == out_dtype else y.to(out_dtype)), ScanState(h_last)


@torch.no_grad()
def gated_scan_chunk(pa: torch.Tensor, px: torch.Tensor, pc1: torch.Tensor, pc2: torch.Tensor, pd: torch.Tensor,
                     state: Optional[ScanState] = None, *, gate_dtype: Optional[torch.dtype] = None,
                     out_dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, ScanState]:
    """``gated.gated_scan`` over one piece ``[B, L_piece, D]`` of a longer sequence; returns ``(y, new_state)``.
    The five projection outputs may be views of one tensor (column slices of a fused projection)."""
    ts = (pa, px, pc1, pc2, pd)
    if any(t.shape != pa.shape for t in ts) or pa.dim() != 3:
        raise ValueError("the five projection outputs must share one shape [B, L, D].")
    if pa.device.type != "cuda":
        raise RuntimeError("gated_scan_chunk requires CUDA tensors.")
    B, L, D = pa.shape
    if state is not None and tuple(state.h.shape) != (B, D):
        raise ValueError(f"state is {tuple(state.h.shape)}, expected {(B, D)}")
    gate_dtype = gate_dtype or pa.dtype
    out_dtype = out_dtype or pa.dtype
    if _fusable(ts, gate_dtype, out_dtype):
        y = torch.empty((B, L, D), dtype=out_dtype, device=pa.device)
        h_last = torch.empty((B, D), dtype=torch.float32, device=pa.device)
        try:
            _lib.gated_scan_fwd(pa, px, pc1, pc2, pd, y, gate_dtype,
                                h_in=None if state is None else state.h.contiguous(), h_last=h_last)
            return y, ScanState(h_last)
        except _lib.Unsupported:
            pass
    a, x, c, b = _gates(pa, px, pc1, pc2, pd, gate_dtype)
    return scan_chunk(x, a, b, c, state, out_dtype=out_dtype)
