"""Products in 8 bits for serving: e4m3 operands with a scale for each block of 128.

    x [..., K]: a scale for each 128 values of a row            ``Fp8Rows``   (``quantize_rows``, ``norm.add_rms_norm_fp8``)
    w [N, K]:   a scale for each 128 x 128 block                ``Fp8Weight`` (``quantize_weight``, once per weight)
    matmul_fp8: y[..., n] = bias[n] + sum over blocks b of sx[..., b] sw[n/128, b] * sum over k in b of x[..., k] w[n, k]

``scale = max(amax, 2^-100) / 448`` and ``value = e4m3(v / scale)``, nearest even; a block with a NaN or an infinity
gives NaN.  Inner sums and the sum over blocks are fp32, the result is rounded once.  ``layers.SSMFp8`` runs an SSM
block on these.  CUDA tensors only; there is no CPU path.  This is a serving path: results never require a gradient."""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

BLOCK = 128
_E4M3 = torch.float8_e4m3fn
_FLOATS = frozenset((torch.float32, torch.float16, torch.bfloat16))


def n_blocks(size: int) -> int:
    return (size + BLOCK - 1) // BLOCK


def rows_2d(t: torch.Tensor) -> torch.Tensor:
    """[..., K] as [rows, K] with a contiguous last axis; copies only where the strides leave no other way."""
    if t.dim() != 2:
        rows = 1
        for n in t.shape[:-1]:
            rows *= n
        t = t.reshape(rows, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


class Fp8Rows:
    """e4m3 ``values`` [..., K] with fp32 ``scales`` [..., ceil(K/128)]."""

    __slots__ = ("values", "scales")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        if values.dtype is not _E4M3 or scales.dtype is not torch.float32:
            raise TypeError(f"values must be float8_e4m3fn and scales float32; got {values.dtype} and {scales.dtype}")
        shape, of = values.shape, scales.shape
        if len(shape) < 1 or len(of) != len(shape) or shape[:-1] != of[:-1] or (shape[-1] + 127) // 128 != of[-1]:
            raise ValueError(f"scales {tuple(scales.shape)} are not one for each 128 of a row of {tuple(values.shape)}")
        self.values, self.scales = values, scales

    @classmethod
    def _of(cls, values: torch.Tensor, scales: torch.Tensor) -> "Fp8Rows":
        """What this package has made itself: nothing to check."""
        q = cls.__new__(cls)
        q.values, q.scales = values, scales
        return q

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    @property
    def device(self) -> torch.device:
        return self.values.device

    def _under(self, shape) -> "Fp8Rows":
        """[rows, K] as the same rows under leading axes ``shape[:-1]``."""
        if len(shape) == 2:
            return self
        if len(shape) == 1:
            return Fp8Rows._of(self.values[0], self.scales[0])
        lead = tuple(shape[:-1])
        return Fp8Rows._of(self.values.unflatten(0, lead), self.scales.unflatten(0, lead))

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        per = self.scales.repeat_interleave(BLOCK, -1)[..., :self.values.shape[-1]]
        return (self.values.float() * per).to(dtype)


class Fp8Weight:
    """e4m3 ``values`` [N, K] with fp32 ``scales`` [ceil(N/128), ceil(K/128)]."""

    __slots__ = ("values", "scales")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        if values.dtype is not _E4M3 or scales.dtype is not torch.float32:
            raise TypeError(f"values must be float8_e4m3fn and scales float32; got {values.dtype} and {scales.dtype}")
        if values.dim() != 2 or scales.shape != ((values.shape[0] + 127) // 128, (values.shape[1] + 127) // 128):
            raise ValueError(f"scales {tuple(scales.shape)} are not one for each 128 x 128 block of {tuple(values.shape)}")
        self.values, self.scales = values, scales

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    @property
    def device(self) -> torch.device:
        return self.values.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        N, K = self.values.shape
        per = self.scales.repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]
        return (self.values.float() * per).to(dtype)


def _values_like(rows: int, K: int, device, dtype: torch.dtype = _E4M3) -> torch.Tensor:
    """e4m3 (or bytes) [rows, K] whose rows start on 16-byte boundaries, as the product's copies need them."""
    return torch.empty_strided((rows, K), ((K + 15) // 16 * 16, 1), dtype=dtype, device=device)


def rows_like(x2: torch.Tensor) -> Fp8Rows:
    """Room for the quantised rows of [rows, K] ``x2``.  The scales lie block by block (all rows of a block side by
    side): 32 rows of a product's tile then read theirs in one access."""
    rows, K = x2.shape
    dev = x2.device
    return Fp8Rows._of(_values_like(rows, K, dev), torch.empty_strided((rows, n_blocks(K)), (1, rows), dtype=torch.float32, device=dev))


def _check_source(x: torch.Tensor, name: str) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"{name} needs CUDA tensors; there is no CPU path")
    if x.dtype not in _FLOATS:
        raise TypeError(f"{name} takes float32, float16 and bfloat16; got {x.dtype}")


def quantize_rows(x: torch.Tensor) -> Fp8Rows:
    """Quantise ``[..., K]`` activations, one scale for each 128 values of a row."""
    _check_source(x, "quantize_rows")
    if x.dim() < 1:
        raise ValueError("quantize_rows takes [..., K]")
    x2 = rows_2d(x)
    q = rows_like(x2)
    _lib.quant_fp8(x2, q.values, q.scales, False)
    return q._under(x.shape)


def quantize_weight(w: torch.Tensor) -> Fp8Weight:
    """Quantise an ``[N, K]`` weight (``torch.nn.Linear`` layout), one scale for each 128 x 128 block."""
    _check_source(w, "quantize_weight")
    if w.dim() != 2:
        raise ValueError("quantize_weight takes an [N, K] weight")
    w2 = rows_2d(w)
    N, K = w2.shape
    q = Fp8Weight(_values_like(N, K, w.device),
                  torch.empty((n_blocks(N), n_blocks(K)), dtype=torch.float32, device=w.device))
    _lib.quant_fp8(w2, q.values, q.scales, True)
    return q


def copyable(values: torch.Tensor):
    """[rows, K] values as the product's copies can address them, and their pitch: a copy where a row or the base is not
    on a 16-byte boundary or the last axis is strided."""
    rows, K = values.shape
    pitch, step = values.stride()
    if (step == 1 or K <= 1) and pitch % 16 == 0 and pitch >= K and values.data_ptr() % 16 == 0:
        return values, pitch
    out = _values_like(rows, K, values.device, values.dtype)
    out.copy_(values)
    return out, out.stride(0)


def matmul_fp8(x: Fp8Rows, w: Fp8Weight, bias: Optional[torch.Tensor] = None, *,
               out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``x @ w.T + bias`` on quantised operands: ``[..., N]`` in ``out_dtype`` (bf16, fp16 or fp32)."""
    xv, xs, wv = x.values, x.scales, w.values
    if not xv.is_cuda:
        raise RuntimeError("matmul_fp8 needs CUDA tensors; there is no CPU path")
    if out_dtype not in _FLOATS:
        raise TypeError(f"out_dtype must be float32, float16 or bfloat16; got {out_dtype}")
    N, K = wv.shape
    *lead, k = xv.shape
    if k != K:
        raise ValueError(f"x has {k} columns, the weight {K}")
    if bias is not None:
        if bias.shape != (N,):
            raise ValueError(f"bias is {tuple(bias.shape)}, expected {(N,)}")
        if bias.dtype not in _FLOATS:
            raise TypeError(f"bias must be float32, float16 or bfloat16; got {bias.dtype}")
        if bias.requires_grad or not bias.is_contiguous():
            bias = bias.detach().contiguous()
    rows = 1
    for n in lead:
        rows *= n
    if len(lead) != 1:
        xv, xs = xv.reshape(rows, K), xs.reshape(rows, xs.shape[-1])
    y = torch.empty_strided((rows, N), (N, 1), dtype=out_dtype, device=xv.device)
    if K == 0:  # an empty sum
        y.copy_(bias) if bias is not None else y.zero_()
    else:
        xv, x_pitch = copyable(xv)
        wv, w_pitch = copyable(wv)
        _lib.matmul_fp8(xv, x_pitch, xs, wv, w_pitch, w.scales, bias, y)
    return y if len(lead) == 1 else y.view(*lead, N)


__all__ = ["BLOCK", "Fp8Rows", "Fp8Weight", "quantize_rows", "quantize_weight", "matmul_fp8"]
