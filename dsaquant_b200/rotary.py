"""Rotary positions on q and k (b200w4a4_rotary) and the tables they read.

`attention_qkv.qk_norm_rope` rotates whole heads in neighbouring pairs, with one table row for each row of its
input.  `apply_rotary` is the form a decoder needs: any position by number, the half or the interleaved layout,
part of the head, q and k (of different head counts, views of a fused projection) in one launch."""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib
from .kernels.vdm_w4a4 import _DTYPE_CODE, _DeviceGuard, _empty, _load_ext, _require_cuda, _stream_ptr

SCALINGS = ("none", "linear", "ntk", "yarn")


def rotary_table(
    max_positions: int,
    rotary_dim: int,
    base: float = 10000.0,
    *,
    scaling: str = "none",
    factor: float = 1.0,
    trained_positions: int = 4096,
    beta_fast: float = 32.0,
    beta_slow: float = 1.0,
    device: Optional[torch.device] = None,
) -> torch.Tensor:
    """fp32 [max_positions, rotary_dim / 2, 2] = (cos, sin) of position p and pair i, computed in 64 bits: what
    `apply_rotary` reads.  With f_i = base^(-2 i / rotary_dim) the angle is p f_i; for contexts longer than the
    trained one
        linear  p f_i / factor
        ntk     f_i of the base base * factor^(rotary_dim / (rotary_dim - 2)): the slowest pair is stretched by factor
        yarn    pairs that turn more than beta_fast times over trained_positions keep f_i, those that turn less than
                beta_slow times get f_i / factor, a linear ramp between; cos and sin are scaled by 0.1 ln(factor) + 1"""
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}")
    if max_positions < 1 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("max_positions must be positive and rotary_dim even")
    if not (base > 1 and factor >= 1 and trained_positions >= 1 and beta_fast > beta_slow > 0):
        raise ValueError("base > 1, factor >= 1, trained_positions >= 1 and beta_fast > beta_slow > 0 are wanted")
    if scaling == "ntk" and rotary_dim == 2:
        raise ValueError("ntk scaling needs a rotary_dim over 2")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
    amplitude = 1.0
    if scaling == "ntk":
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = base ** (-2.0 * i / rotary_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        def pair_of(turns: float) -> float:  # the pair that turns so often over the trained positions
            return rotary_dim * math.log(trained_positions / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f * (1 - ramp) + f / factor * ramp
        amplitude = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * f
    return (torch.stack([angle.cos(), angle.sin()], -1) * amplitude).float()


def _check_rows(x: torch.Tensor, name: str, like: Optional[torch.Tensor]) -> None:
    if x.dim() != 3 or (x.shape[2] > 1 and x.stride(2) != 1):
        raise ValueError(f"{name} must be [T, heads, head_dim] with unit stride in the head")
    if like is not None and (x.shape[0] != like.shape[0] or x.shape[2] != like.shape[2] or x.dtype != like.dtype
                             or x.device != like.device):
        raise ValueError(f"{name} must match q in tokens, head_dim, dtype and device")


def apply_rotary(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    cos_sin: torch.Tensor,
    positions: torch.Tensor,
    *,
    interleaved: bool = False,
    inverse: bool = False,
    inplace: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q [T, q_heads, head_dim] and k [T, k_heads, head_dim] (or None), fp16, bf16 or fp32, rotated by the rows
    `positions` (int32 or int64 [T]) of cos_sin, a table as `rotary_table` makes it; its second dimension says how much
    of the head is rotated, the rest is copied.  Token and head strides are free.  interleaved: pairs (2i, 2i + 1)
    instead of (i, i + rotary_dim / 2).  inverse: rotates back (the transpose; also the gradient).
    Returns new contiguous tensors, or with inplace the given ones, overwritten.
    A token at a negative position (padding) is copied unchanged; one behind the table comes out as NaN."""
    lib = _load_ext()
    _require_cuda(q, "q")
    if q.dtype not in _DTYPE_CODE:
        raise RuntimeError("apply_rotary takes float16, bfloat16 or float32")
    _check_rows(q, "q", None)
    if k is not None:
        _check_rows(k, "k", q)
    dev = q.device
    t, hq, hd = q.shape
    hk = k.shape[1] if k is not None else 0
    if cos_sin.dim() != 3 or cos_sin.shape[2] != 2 or cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous():
        raise ValueError("cos_sin must be a contiguous float32 [positions, rotary_dim / 2, 2] table")
    rd = 2 * cos_sin.shape[1]
    if cos_sin.shape[0] < 1 or not 2 <= rd <= hd or hd > 512:
        raise ValueError("the table must rotate between 2 and head_dim (at most 512) values")
    if positions.dtype not in (torch.int32, torch.int64) or positions.dim() != 1 or positions.shape[0] != t:
        raise ValueError("positions must be int32 or int64 with one value for each token")
    if cos_sin.device != dev or positions.device != dev:
        raise ValueError("q, cos_sin and positions must be on one device")
    if hq < 1 or (k is not None and hk < 1):
        raise ValueError("q and k must have heads")
    if inplace:
        q_out, k_out = q, k
    else:
        q_out = _empty((t, hq, hd), q.dtype, dev)
        k_out = _empty((t, hk, hd), q.dtype, dev) if k is not None else None
    if t > 0:
        pos = positions if positions.is_contiguous() else positions.contiguous()
        qs, qos = q.stride(), q_out.stride()
        ks, kos = (k.stride(), k_out.stride()) if k is not None else ((0, 0), (0, 0))
        with _DeviceGuard(dev):
            rc = lib.b200w4a4_rotary(
                q.data_ptr(), qs[0], qs[1], q_out.data_ptr(), qos[0], qos[1], hq, k.data_ptr() if k is not None else None,
                ks[0], ks[1], k_out.data_ptr() if k is not None else None, kos[0], kos[1], hk, _DTYPE_CODE[q.dtype],
                cos_sin.data_ptr(), cos_sin.shape[0], pos.data_ptr(), 1 if pos.dtype == torch.int64 else 0, t, hd, rd,
                1 if interleaved else 0, 1 if inverse else 0, _stream_ptr(dev))
        _lib.check(rc, "rotary")
    return q_out, k_out
