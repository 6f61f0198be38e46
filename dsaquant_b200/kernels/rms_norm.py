"""Residual addition, RMSNorm and per-token 8-bit codes in one kernel (b200w4a4_rms_norm_quant): what stands
between the residual stream of a decoder layer and its 4-bit linears.  The int8 codes and fp32 scales are those
`vdm_w4a4.linear_prequantized` (prompts) and `w4_group.linear_w4_group` (single tokens) take; the e4m3 form is for
fp8 products.  CUDA only, on the current stream, nothing is kept between calls."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _lib
from .vdm_w4a4 import _DTYPE_CODE, _empty, _load_ext, _require_cuda, _run, _stream_ptr

_FORMATS = {torch.int8: 0, torch.float8_e4m3fn: 1}
MAX_WIDTH = 16384


def _rows(x: torch.Tensor, d: int) -> torch.Tensor:
    """x as [rows, d] with unit column stride; a view wherever the rows have one pitch."""
    x2 = x if x.dim() == 2 else x.reshape(-1, d)
    if (d > 1 and x2.stride(1) != 1) or (x2.shape[0] > 1 and x2.stride(0) < d):
        x2 = x2.contiguous()
    return x2


def rms_norm_quant(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
    *,
    residual: Optional[torch.Tensor] = None,
    out_dtype: torch.dtype = torch.int8,
    clip_ratio: float = 1.0,
) -> Tuple[torch.Tensor, ...]:
    """x [..., D] (fp16, bf16 or fp32), weight [D] -> (codes [..., D] of out_dtype, scale fp32 [...]), and with a
    residual of x's shape and type also the new residual stream (x + residual rounded once to that type).

        s = x + residual;  y = s * rsqrt(mean(s^2) + eps) * weight
        scale = max(max|y|, 1e-5) / top * clip_ratio      top = 127 for torch.int8, 448 for torch.float8_e4m3fn
        codes = clamp(rint(y / scale), -128, 127)         or y / scale rounded to e4m3, saturating

    Everything is fp32 and reads s before its rounding: int8 codes are those of the fp32 quotient by the scale that is returned,
    e4m3 codes those of the exact quotient (values beside a border are decided in 64 bits).  D is at most 16384.  Rows may be strided (views of a
    wider tensor are read in place).  A row whose sum of squares is not finite in fp32 (it
    holds an infinity, a NaN, or values near 1e19), whose mean square and eps add up to less than fp32's normal range (values
    below 1e-19 with an eps of 0), or whose scale leaves 1.2e-38 .. 8.5e37 has scale NaN and codes 0.  Forward only, as every operator here."""
    lib = _load_ext()
    _require_cuda(x, "x")
    if x.dtype not in _DTYPE_CODE or weight.dtype not in _DTYPE_CODE:
        raise RuntimeError("rms_norm_quant takes float16, bfloat16 or float32")
    if out_dtype not in _FORMATS:
        raise ValueError("out_dtype must be int8 or float8_e4m3fn")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"the last dimension of x must have 1 to {MAX_WIDTH} elements")
    d = x.shape[-1]
    dev = x.device
    if weight.device != dev or weight.dim() != 1 or weight.shape[0] != d:
        raise ValueError("weight must be a [D] vector on x's device")
    if not (clip_ratio > 0 and eps >= 0):
        raise ValueError("clip_ratio must be positive and eps not negative")
    r2 = stream_out = None
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != dev:
            raise ValueError("residual must have x's shape, dtype and device")
        r2 = _rows(residual, d)
        stream_out = _empty(x.shape, x.dtype, dev)
    x2 = _rows(x, d)
    m = x2.shape[0]
    if m >= 1 << 31:
        raise ValueError("x must have fewer than 2^31 rows")
    w = weight if weight.is_contiguous() else weight.contiguous()
    codes = _empty(x.shape, out_dtype, dev)
    scale = _empty(x.shape[:-1], torch.float32, dev)
    if m > 0:
        rc = _run(
            dev, lib.b200w4a4_rms_norm_quant, x2.data_ptr(), _DTYPE_CODE[x.dtype], x2.stride(0) if m > 1 else d,
            r2.data_ptr() if r2 is not None else None, r2.stride(0) if r2 is not None and m > 1 else d, w.data_ptr(),
            _DTYPE_CODE[w.dtype], float(eps), codes.data_ptr(), _FORMATS[out_dtype], scale.data_ptr(),
            stream_out.data_ptr() if stream_out is not None else None, m, d, float(clip_ratio), _stream_ptr(dev))
        _lib.check(rc, "rms_norm_quant")
    return (codes, scale) if residual is None else (codes, scale, stream_out)
