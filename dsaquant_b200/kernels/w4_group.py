"""4-bit weights with group scales for a few tokens (b200w4a4_linear_w4_group): the single-token companion of
`vdm_w4a4.linear_vdm_w4a4`, whose GEMM works on tiles of 256 tokens and per-channel scales.

A weight is two tensors, usable as they are (nothing is laid out or kept for it):
    packed  uint8 [N, K/2]        code 2b in the low and 2b + 1 in the high nibble of byte b, two's complement
    scales  float16 [N, K/group]  one for every `group` consecutive codes of a row (a multiple of 32)
The weights of that GEMM (vdm_w4a4_packed_v1: the buffers of QuantLinear and of packed checkpoints) have the same types and,
for groups of 64, the same shapes, but their codes and scales lie in the order of its tiles.  `regroup_packed_weight` turns one
into the form used here, with the same codes and scales; the tensors that this package makes, loads or has used as
such weights are refused (a copy that a program makes of one by hand is not known as one).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _lib
from .vdm_w4a4 import _DTYPE_CODE, _empty, _load_ext, _require_cuda, _run, _stream_ptr, in_gemm_layout, unpack_codes

_X_CODE = {torch.float16: 0, torch.bfloat16: 1, torch.int8: 3}
MAX_TOKENS = 65535 * 8
MAX_ROWS, MAX_WIDTH = (1 << 31) - 512, 1 << 20  # of the weight (the foreign calls take 32-bit sizes)
_OUT_CODE = {torch.float16: 0, torch.bfloat16: 1}
_BIAS_F32 = 16


def quantize_weight_grouped(weight: torch.Tensor, group_size: int = 128) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp weight [N, K] -> (packed, scales): scale = max(absmax, 1e-5) / 7 of each group in fp16,
    code = clamp(rint(w / scale), -8, 7).  A group that holds a NaN or an infinity, or a value past 458000 (its scale would
    pass fp16's range), has scale NaN and codes 0: outputs of that row are NaN."""
    lib = _load_ext()
    _require_cuda(weight, "weight")
    if weight.dtype not in _DTYPE_CODE or weight.dim() != 2:
        raise RuntimeError("weight must be a float16, bfloat16 or float32 [N, K] matrix")
    n, k = weight.shape
    if n < 1 or group_size < 32 or group_size % 32 or k < 1 or k % group_size:
        raise ValueError("group_size must be a multiple of 32 that divides K")
    if n > MAX_ROWS or k > MAX_WIDTH:
        raise ValueError(f"a weight has at most {MAX_ROWS} rows of {MAX_WIDTH} values")
    w = weight.detach().contiguous()
    packed = torch.empty((n, k // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((n, k // group_size), dtype=torch.float16, device=w.device)
    rc = _run(w.device, lib.b200w4a4_quantize_weight_grouped, w.data_ptr(), _DTYPE_CODE[w.dtype], packed.data_ptr(),
              scales.data_ptr(), n, k, group_size, _stream_ptr(w.device))
    _lib.check(rc, "quantize_weight_grouped")
    return packed, scales


def regroup_packed_weight(qweight: torch.Tensor, channel_scales: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """vdm_w4a4_packed_v1 codes [N, K/2] and their plain per-channel scales fp16 [N] (`vdm_weight_packed` and
    `vdm_weight_scale` of a layer, the first and third result of `quantize_weight_per_channel`) -> (packed, scales [N, 1]): the
    same weight with one group a row, for prompts through the GEMM and tokens through `linear_w4_group`."""
    _require_cuda(qweight, "qweight")
    n, k = qweight.shape[0], 2 * qweight.shape[1]
    if qweight.dtype != torch.uint8 or qweight.dim() != 2 or n % 128 or k % 64 or n * k == 0:
        raise ValueError("qweight must be uint8 [N, K/2] with N a multiple of 128 and K one of 64")
    if channel_scales.dtype != torch.float16 or channel_scales.shape != (n,) or channel_scales.device != qweight.device:
        raise ValueError("channel_scales must be float16 [N] on qweight's device")
    codes = unpack_codes(qweight, n, k, 2).view(torch.uint8)
    return codes[:, 0::2].bitwise_and(15) | codes[:, 1::2] << 4, channel_scales.detach().clone().unsqueeze(1)


def linear_w4_group(
    x: torch.Tensor,
    packed: torch.Tensor,
    scales: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    *,
    act_scale: Optional[torch.Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """x [..., K] times the grouped 4-bit weight, plus bias [N]: [..., N].  x is fp16 or bf16 (multiplied as it is,
    fp32 sums), or int8 codes with act_scale, their fp32 scale per token, as `rms_norm_quant` and
    `quantize_activation_per_token` return them.  out_dtype: fp16 or bf16, by default x's (fp16 for int8).  The bias is
    added in fp32, whatever its type, before the one rounding to out_dtype.
    For single tokens and small batches: the weight is read once for every 8 to 32 tokens, and any number of
    tokens is right, but from some hundreds on a GEMM is faster."""
    lib = _load_ext()
    _require_cuda(x, "x")
    if x.dtype not in _X_CODE:
        raise RuntimeError("x must be float16, bfloat16 or int8")
    if packed.dtype != torch.uint8 or scales.dtype != torch.float16 or packed.dim() != 2 or scales.dim() != 2:
        raise RuntimeError("packed must be uint8 [N, K/2] and scales float16 [N, K/group]")
    if in_gemm_layout(packed) or in_gemm_layout(scales):
        raise ValueError("this weight lies in the GEMM's order (vdm_w4a4_packed_v1): regroup_packed_weight makes a grouped one of it")
    n, k = packed.shape[0], packed.shape[1] * 2
    groups = scales.shape[1]
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"the last dimension of x must be K={k}")
    if n < 1 or k < 1 or scales.shape[0] != n or groups < 1 or k % groups or (k // groups) % 32:
        raise ValueError("scales must be [N, K/group] with a group that is a multiple of 32 and divides K")
    if n > MAX_ROWS or k > MAX_WIDTH:
        raise ValueError(f"a weight has at most {MAX_ROWS} rows of {MAX_WIDTH} values")
    dev = x.device
    if packed.device != dev or scales.device != dev:
        raise ValueError("x, packed and scales must be on one device")
    if out_dtype is None:
        out_dtype = torch.float16 if x.dtype == torch.int8 else x.dtype
    if out_dtype not in _OUT_CODE:
        raise ValueError("out_dtype must be float16 or bfloat16")
    x2 = x if x.dim() == 2 else x.reshape(-1, k)
    if not x2.is_contiguous() or x2.data_ptr() % 16:
        x2 = x2.clone(memory_format=torch.contiguous_format)
    m = x2.shape[0]
    if m > MAX_TOKENS:
        raise ValueError(f"at most {MAX_TOKENS} tokens a call")
    if not packed.is_contiguous() or packed.data_ptr() % 16 or not scales.is_contiguous():
        raise ValueError("packed (16-byte aligned) and scales must be contiguous")
    if (act_scale is not None) != (x.dtype == torch.int8):
        raise ValueError("act_scale goes with int8 codes, and only with them")
    if act_scale is not None:
        if act_scale.dtype != torch.float32 or act_scale.numel() != m or act_scale.device != dev:
            raise ValueError("act_scale must be float32 with one value for each token")
        act_scale = act_scale.contiguous()
    out_code = _OUT_CODE[out_dtype]
    if bias is not None:
        if bias.numel() != n or bias.device != dev:
            raise ValueError("bias must have N elements")
        if bias.dtype != out_dtype:  # added before the one rounding to the output's type, as it is
            bias = bias.float()
            out_code |= _BIAS_F32
        bias = bias.contiguous()
    out = _empty((*x.shape[:-1], n), out_dtype, dev)
    if m > 0:
        rc = _run(
            dev, lib.b200w4a4_linear_w4_group, x2.data_ptr(), _X_CODE[x.dtype],
            act_scale.data_ptr() if act_scale is not None else None, packed.data_ptr(), scales.data_ptr(),
            bias.data_ptr() if bias is not None else None, out.data_ptr(), out_code, m, n, k, k // groups,
            _stream_ptr(dev))
        _lib.check(rc, "linear_w4_group")
    return out
