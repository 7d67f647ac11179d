"""RMS normalisation of the layer input as one kernel per direction.

``rms_norm(x, weight, eps)`` computes what ``layers.RMSNorm`` computes
(reference: quick_ssm/layers.py:9-17), ``x * weight / sqrt(mean(x^2, -1) + eps)``, through
``qssm_rmsnorm_fwd`` / ``qssm_rmsnorm_bwd``: the forward reads x and writes y, the backward reads x
and dy and writes dx; dw is summed in a fixed order (no atomics).  Shapes the kernels cannot take
(last axis not a multiple of 4, unaligned views) are composed from torch operations on the same
device; CPU tensors raise.

``add_rms_norm`` and ``add_rms_norm_fp8`` put the residual's addition in front, as it stands between
two blocks of a stack: ``h = x + residual`` is written once and its norm leaves the same kernel, in
x's type with a backward pass (training), or in e4m3 with a scale for each 128 values (serving, the
operand of ``fp8.matmul_fp8``).  They take any row length, pitch and alignment.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .fp8 import Fp8Rows, rows_2d, rows_like


def _composed(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    norm = torch.sqrt(x.pow(2).mean(dim=-1, keepdim=True) + eps)
    return x * (weight / norm)


class _RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        xc = x.contiguous()
        w32 = weight.detach().float().contiguous()
        y = torch.empty_like(xc)
        rows = xc.numel() // xc.shape[-1] if xc.shape[-1] else 0
        rstd = torch.empty(rows, dtype=torch.float32, device=xc.device)
        _lib.rmsnorm_fwd(xc, w32, y, rstd, eps)
        ctx.save_for_backward(xc, w32, rstd)
        ctx.w_dtype = weight.dtype
        return y

    @staticmethod
    def backward(ctx, dy):
        xc, w32, rstd = ctx.saved_tensors
        dyc = dy.contiguous()
        if dyc.dtype != xc.dtype:
            dyc = dyc.to(xc.dtype)
        dx = torch.empty_like(xc)
        dw = torch.empty_like(w32)
        _lib.rmsnorm_bwd(xc, w32, dyc, rstd, dx, dw)
        return dx, dw.to(ctx.w_dtype), None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    if x.device.type != "cuda":
        raise RuntimeError("rms_norm needs CUDA tensors; there is no CPU path")
    if weight.shape != x.shape[-1:]:
        raise ValueError("weight must have the size of the last axis of x")
    H = x.shape[-1]
    if H % 4 != 0 or x.numel() == 0 or x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        return _composed(x, weight, eps)
    return _RMSNormFunction.apply(x, weight, eps)


FLOATS = frozenset((torch.float32, torch.float16, torch.bfloat16))


def _check_add(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, name: str) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"{name} needs CUDA tensors; there is no CPU path")
    dt, shape = x.dtype, x.shape
    if dt not in FLOATS or weight.dtype not in FLOATS:
        raise TypeError(f"{name} takes float32, float16 and bfloat16; got {dt} with a weight in {weight.dtype}")
    if len(shape) < 1 or weight.shape != shape[-1:]:
        raise ValueError("weight must have the size of the last axis of x")
    if residual is not None:
        if residual.shape != shape:
            raise ValueError(f"residual is {tuple(residual.shape)}, x is {tuple(shape)}")
        if residual.dtype is not dt and residual.dtype is not torch.float32:
            raise TypeError(f"residual must be in x's type or in float32; got {residual.dtype} with x in {dt}")


def _room_like(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """An uninitialised tensor of t's shape whose rows lie one behind the other (``empty_like`` takes half of ``empty``'s
    time on the host).  Left to itself ``empty_like`` keeps t's strides, and those of axes of size 1 may be anything."""
    if t.dtype is dtype:
        return torch.empty_like(t, memory_format=torch.contiguous_format)
    return torch.empty(t.shape, dtype=dtype, device=t.device)


class _AddRMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        x2, r2, w = rows_2d(x), rows_2d(residual), weight.contiguous()
        y = _room_like(x, x.dtype)
        h = _room_like(residual, residual.dtype)
        rstd = torch.empty_strided((x2.shape[0],), (1,), dtype=torch.float32, device=x.device) \
            if any(ctx.needs_input_grad) else None
        _lib.add_rmsnorm_fwd(x2, r2, w, rows_2d(y), rows_2d(h), rstd, eps)
        if rstd is not None:
            ctx.save_for_backward(h, w, rstd)
            ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        if torch.is_grad_enabled():
            raise RuntimeError("add_rms_norm has no second derivative")
        h, w, rstd = ctx.saved_tensors
        need_x, need_r, need_w, _ = ctx.needs_input_grad
        if dy is None:  # only h was used: its gradient passes through
            return (dh if need_x else None), (dh if need_r else None), None, None
        # autograd hands over gradients in the outputs' types and takes the inputs' own back
        xd, rd = dy.dtype, h.dtype
        dx = _room_like(h, xd) if need_x or rd is xd else None
        dres = _room_like(h, rd) if rd is not xd and (need_r or dx is None) else None
        dw = torch.empty_like(w)
        _lib.add_rmsnorm_bwd(rows_2d(h), w, rows_2d(dy), None if dh is None else rows_2d(dh), rstd,
                             None if dx is None else rows_2d(dx), None if dres is None else rows_2d(dres), dw)
        return (dx if need_x else None), ((dx if rd is xd else dres) if need_r else None), (dw if need_w else None), None


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                 eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """``h = x + residual`` and ``y = h * weight / sqrt(mean(h^2, -1) + eps)``; returns ``(y, h)``.

    ``x``: ``[..., H]`` fp32, fp16 or bf16; ``residual``: the same shape, in x's type or in fp32 (a 32-bit residual
    stream under 16-bit branches).  ``y`` has x's type, ``h`` the residual's; the norm is that of ``h`` as stored.
    Differentiable (once) in x, residual and weight."""
    if residual is None:
        raise ValueError("add_rms_norm needs a residual; rms_norm is the norm alone")
    _check_add(x, residual, weight, "add_rms_norm")
    return _AddRMSNormFunction.apply(x, residual, weight, float(eps))


def add_rms_norm_fp8(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor,
                     eps: float = 1e-5) -> Tuple[Fp8Rows, torch.Tensor]:
    """The sum and norm of ``add_rms_norm`` with y quantised for ``fp8.matmul_fp8``; returns ``(y, h)``.

    The scales are taken from y in 32 bits: it is rounded once, to e4m3.  ``residual=None`` (the first block of a
    stack): h is x itself.  Serving only, no gradient."""
    _check_add(x, residual, weight, "add_rms_norm_fp8")
    x2 = rows_2d(x)
    q = rows_like(x2)
    w = weight.contiguous()
    if residual is None:
        h = x
        _lib.add_rmsnorm_fp8(x2, None, w, q.values, q.scales, None, float(eps))
    else:
        h = _room_like(residual, residual.dtype)
        _lib.add_rmsnorm_fp8(x2, rows_2d(residual), w, q.values, q.scales, rows_2d(h), float(eps))
    return q._under(x.shape), h
