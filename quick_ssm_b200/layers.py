"""Caller of the scan: the gated SSM block and its RMS norm, with the constructor and forward
signatures of the reference's ``quick_ssm/layers.py`` (``RMSNorm`` :9-17, ``SSM`` :20-107) so
that the reference's training and example scripts run against this package unchanged.  The
projections stay in torch (cuBLAS GEMMs); only the scan goes through the CUDA library."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from .scan_interface import scan


class RMSNorm(nn.Module):
    def __init__(self, hidden_size: int, eps: float = 1e-5, dtype=torch.float32, device=None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(hidden_size, dtype=dtype, device=device))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        rms = torch.sqrt(x.pow(2).mean(dim=-1, keepdim=True) + self.eps)
        return x * (self.weight / rms)


class RMSNormFused(RMSNorm):
    """``RMSNorm`` through the normalisation kernels (``norm.rms_norm``): same parameter, same
    result up to fp32 rounding, one kernel per direction instead of torch's element-wise chain."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.device.type != "cuda":
            return super().forward(x)
        from .norm import rms_norm
        return rms_norm(x, self.weight, self.eps)


class SSM(nn.Module):
    """Pre-norm, five input projections (decay, input, two halves of a SwiGLU output gate, input
    gate), the scan over the state dimension, output projection, residual."""

    def __init__(self, hidden_size: int, state_size_mult: float = 1.0, eps: float = 1e-5,
                 dtype: torch.dtype = torch.float32, device: Optional[torch.device] = None,
                 compute_dtype: torch.dtype = torch.float16, use_residual: bool = True, use_norm: bool = True):
        super().__init__()
        self.hidden_size = hidden_size
        self.state_size_dim = int(hidden_size * state_size_mult)
        self.compute_dtype = compute_dtype
        self.use_residual = use_residual
        self.use_norm = use_norm
        kw = dict(device=device, dtype=dtype)
        n = self.state_size_dim
        self.A_proj = nn.Linear(hidden_size, n, bias=True, **kw)
        self.B_proj = nn.Linear(hidden_size, n, bias=False, **kw)
        self.C_proj_a = nn.Linear(hidden_size, n, bias=False, **kw)
        self.C_proj_b = nn.Linear(hidden_size, n, bias=False, **kw)
        self.D_proj = nn.Linear(hidden_size, n, bias=False, **kw)
        self.out_proj = nn.Linear(n, hidden_size, bias=True, **kw)
        self.pre_norm = RMSNorm(hidden_size, eps=eps, dtype=dtype, device=device) if use_norm else nn.Identity()

    def forward(self, x: torch.Tensor, *, block_l: int = 256, checkpoint: bool = True,
                tile_b: Optional[int] = None, tile_d: Optional[int] = None, backend: str = "auto",
                scan_out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        skip = x if self.use_residual else 0
        u = self.pre_norm(x) if self.use_norm else x
        cd = self.compute_dtype
        decay = torch.sigmoid(self.A_proj(u)).to(cd)
        drive = self.B_proj(u).to(cd)
        out_gate = (F.silu(self.C_proj_a(u)) * self.C_proj_b(u)).to(cd)
        in_gate = torch.sigmoid(self.D_proj(u)).to(cd)
        if scan_out_dtype is None:
            scan_out_dtype = self.out_proj.weight.dtype
        h = scan(x=drive, a=decay, b=in_gate, c=out_gate, block_l=block_l, checkpoint=checkpoint,
                 tile_b=tile_b, tile_d=tile_d, out_dtype=scan_out_dtype, backend=backend)
        return self.out_proj(h.to(self.out_proj.weight.dtype)) + skip


class SSMFused(SSM):
    """``SSM`` with the gate activations fused into the scan kernels (``gated.gated_scan``) and the
    pre-norm done by the normalisation kernels (``norm.rms_norm``): same parameters, same arguments,
    same result up to the rounding of the activations; the element-wise kernels around the
    projections, and their backward, disappear."""

    def forward(self, x: torch.Tensor, *, block_l: int = 256, checkpoint: bool = True,
                tile_b: Optional[int] = None, tile_d: Optional[int] = None, backend: str = "auto",
                scan_out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        if backend == "torch" or x.device.type != "cuda" or not checkpoint:
            return super().forward(x, block_l=block_l, checkpoint=checkpoint, tile_b=tile_b, tile_d=tile_d,
                                   backend=backend, scan_out_dtype=scan_out_dtype)
        skip = x if self.use_residual else 0
        return self._branch(self._normed(x) if self.use_norm else x, scan_out_dtype) + skip

    def _normed(self, x: torch.Tensor) -> torch.Tensor:
        """The normalisation kernels on the layer's own weight.  They keep x's type, where the plain norm's product promotes x
        to the weight's: so does this one where the projections are in another type than x and autocast does not see to it."""
        from .norm import rms_norm
        w = self.pre_norm.weight
        if x.dtype != self.out_proj.weight.dtype and not torch.is_autocast_enabled("cuda"):
            x = x.to(torch.promote_types(x.dtype, w.dtype))
        return rms_norm(x, w, self.pre_norm.eps)

    def _branch(self, u: torch.Tensor, scan_out_dtype: Optional[torch.dtype]) -> torch.Tensor:
        """The block behind its pre-norm and in front of its residual."""
        from .gated import gated_scan
        if scan_out_dtype is None:
            scan_out_dtype = self.out_proj.weight.dtype
        h = gated_scan(self.A_proj(u), self.B_proj(u), self.C_proj_a(u), self.C_proj_b(u), self.D_proj(u),
                       gate_dtype=self.compute_dtype, out_dtype=scan_out_dtype)
        return self.out_proj(h.to(self.out_proj.weight.dtype))


class SSMStack(nn.Module):
    """``n_layers`` residual SSM blocks, the same function as ``nn.Sequential`` of ``SSM`` with the same weights.
    The residual stream and the blocks' outputs are kept apart between two blocks, so that the residual's addition and
    the next block's norm are one kernel per direction (``norm.add_rms_norm``); on the CPU, without ``checkpoint`` and in
    float64 the blocks run one after the other.  ``layers`` holds the blocks; a state dict of such a ``Sequential`` loads with
    its keys prefixed by ``layers.``.  Hooks are called on the projections, not on the blocks and their norms."""

    def __init__(self, n_layers: int, hidden_size: int, state_size_mult: float = 1.0, eps: float = 1e-5,
                 dtype: torch.dtype = torch.float32, device: Optional[torch.device] = None,
                 compute_dtype: torch.dtype = torch.float16):
        super().__init__()
        self.layers = nn.ModuleList(SSMFused(hidden_size, state_size_mult, eps, dtype, device, compute_dtype)
                                    for _ in range(n_layers))

    def forward(self, x: torch.Tensor, *, block_l: int = 256, checkpoint: bool = True,
                tile_b: Optional[int] = None, tile_d: Optional[int] = None, backend: str = "auto",
                scan_out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        from .norm import FLOATS, add_rms_norm
        if (backend == "torch" or x.device.type != "cuda" or not checkpoint or not self.layers or x.dtype not in FLOATS
                or self.layers[0].out_proj.weight.dtype not in FLOATS):
            for layer in self.layers:
                x = layer(x, block_l=block_l, checkpoint=checkpoint, tile_b=tile_b, tile_d=tile_d, backend=backend,
                          scan_out_dtype=scan_out_dtype)
            return x
        first = self.layers[0]
        h, y = x, first._branch(first._normed(x), scan_out_dtype)
        for layer in self.layers[1:]:
            if h.dtype not in (y.dtype, torch.float32):  # as their sum would be promoted
                h = h.float()
            u, h = add_rms_norm(y, h, layer.pre_norm.weight, layer.pre_norm.eps)
            y = layer._branch(u, scan_out_dtype)
        return y + h


class SSMFp8(nn.Module):
    """An ``SSM`` block for serving, its projections in 8 bits (``fp8.matmul_fp8``): made from a trained block with
    ``SSMFp8(block)``.  One pass is five kernels for a prompt and for a single token alike: residual sum, norm and
    quantisation; the five input projections as one product; the scan with its gates and a carried state; quantisation;
    the output projection.  A state size whose bytes in ``act_dtype`` are no multiple of 16 cannot be sliced for the fused
    scan: its gates are torch's element-wise kernels then.  No gradient.

    ``forward(x, residual, state)`` takes the previous block's output and the residual stream apart (``residual=None``:
    x is the stream itself) and returns ``(out, residual, state)``; the stream behind this block is ``out + residual``.
    ``state`` is a ``streaming.ScanState`` or None at the start of a sequence.

    Gates are held in ``gate_dtype`` (the block's compute type, bfloat16 for a float32 one), projections, the scan's output
    and ``out`` in ``act_dtype``: that type too, but float32 for float16 gates of a block whose weights are wider.  The block
    holds these three in its weights' type, and what lies beyond float16's 65504 there is finite here as well."""

    def __init__(self, block: SSM, gate_dtype: Optional[torch.dtype] = None):
        super().__init__()
        if not (block.use_norm and block.use_residual):
            raise ValueError("SSMFp8 serves blocks with a pre-norm and a residual")
        if block.A_proj.weight.device.type != "cuda":
            raise RuntimeError("SSMFp8 needs a block on a CUDA device; there is no CPU path")
        from .fp8 import quantize_weight
        n = block.state_size_dim
        self.state_size_dim, self.hidden_size, self.eps = n, block.hidden_size, block.pre_norm.eps
        if gate_dtype is None:
            gate_dtype = block.compute_dtype if block.compute_dtype != torch.float32 else torch.bfloat16
        if gate_dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"gates are bfloat16 or float16; got {gate_dtype}")
        self.gate_dtype = self.act_dtype = gate_dtype
        if gate_dtype == torch.float16 and block.out_proj.weight.dtype != torch.float16:
            self.act_dtype = torch.float32
        with torch.no_grad():
            w_in = quantize_weight(torch.cat([m.weight for m in (block.A_proj, block.B_proj, block.C_proj_a,
                                                                 block.C_proj_b, block.D_proj)]))
            w_out = quantize_weight(block.out_proj.weight)
            bias = torch.zeros(5 * n, dtype=torch.float32, device=block.A_proj.weight.device)
            bias[:n] = block.A_proj.bias
            self._keep("in", w_in, bias)
            self._keep("out", w_out, block.out_proj.bias.detach().float().clone())
            self.register_buffer("norm_weight", block.pre_norm.weight.detach().clone())

    def _keep(self, name: str, w, bias: torch.Tensor) -> None:
        # bytes: the values' rows are spaced for the copy engine, and a state dict keeps them as they are
        self.register_buffer(f"{name}_values", w.values.view(torch.uint8))
        self.register_buffer(f"{name}_scales", w.scales)
        self.register_buffer(f"{name}_bias", bias)

    def _space(self) -> None:
        """Space the values' rows again where a move or a state dict has closed them up, once and not in every call."""
        from .fp8 import copyable
        for name in ("in_values", "out_values"):
            setattr(self, name, copyable(getattr(self, name))[0])

    def _apply(self, fn, recurse: bool = True):
        super()._apply(fn, recurse)
        self._space()
        return self

    def _load_from_state_dict(self, *args, **kwargs):
        super()._load_from_state_dict(*args, **kwargs)
        self._space()

    def _weight(self, name: str):
        from .fp8 import Fp8Weight
        return Fp8Weight(getattr(self, f"{name}_values").view(torch.float8_e4m3fn), getattr(self, f"{name}_scales"))

    @torch.no_grad()
    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None, state=None):
        from .fp8 import matmul_fp8, quantize_rows
        from .norm import add_rms_norm_fp8
        from .streaming import gated_scan_chunk
        if residual is not None and residual.dtype not in (x.dtype, torch.float32):  # as their sum would be promoted
            residual = residual.float()
        u, h = add_rms_norm_fp8(x, residual, self.norm_weight, self.eps)
        p = matmul_fp8(u, self._weight("in"), self.in_bias, out_dtype=self.act_dtype)
        y, state = gated_scan_chunk(*p.split(self.state_size_dim, dim=-1), state, gate_dtype=self.gate_dtype)
        out = matmul_fp8(quantize_rows(y), self._weight("out"), self.out_bias, out_dtype=self.act_dtype)
        return out, h, state


class SSMStackFp8(nn.Module):
    """A stack of ``SSM`` blocks (an ``SSMStack``, or any iterable of blocks) for serving in 8 bits.
    ``forward(x, states)`` feeds ``[B, L, hidden]`` (a prompt, or the next token with ``L = 1``) and returns
    ``(y, states)``: y in x's type, the states to pass with the next piece."""

    def __init__(self, blocks, gate_dtype: Optional[torch.dtype] = None):
        super().__init__()
        self.layers = nn.ModuleList(SSMFp8(b, gate_dtype) for b in getattr(blocks, "layers", blocks))

    @torch.no_grad()
    def forward(self, x: torch.Tensor, states=None):
        if states is None:
            states = [None] * len(self.layers)
        if len(states) != len(self.layers):
            raise ValueError(f"{len(states)} states for {len(self.layers)} blocks")
        if not self.layers:
            return x, []
        if x.dim() != 3:
            raise ValueError("x must be [B, L, hidden]")
        y, h, after = x, None, []
        for layer, state in zip(self.layers, states):
            y, h, state = layer(y, h, state)
            after.append(state)
        return (h + y).to(x.dtype), after


__all__ = ["SSM", "SSMFused", "SSMStack", "SSMFp8", "SSMStackFp8", "RMSNorm", "RMSNormFused"]
