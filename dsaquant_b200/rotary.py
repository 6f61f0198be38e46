"""Rotary positions on q and k (b200w4a4_rotary) and the tables they read.

`attention_qkv.qk_norm_rope` rotates whole heads in neighbouring pairs, with one table row for each row of its
input.  `apply_rotary` is the form a decoder needs: any position by number, the half or the interleaved layout,
part of the head, q and k (of different head counts, views of a fused projection) in one launch."""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib
from .kernels.vdm_w4a4 import _DTYPE_CODE, _empty, _load_ext, _require_cuda, _run, _stream_ptr

MAX_HEADS = 65536
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
        # where the clamps moved an end of the ramp (a short trained length, a slow base): no pair on its wrong side
        turns = trained_positions * f / (2 * math.pi)
        ramp = torch.where(turns < beta_slow, 1.0, torch.where(turns > beta_fast, 0.0, ramp))
        f = f * (1 - ramp) + f / factor * ramp
        amplitude = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * f
    return (torch.stack([angle.cos(), angle.sin()], -1) * amplitude).float()


def _distinct(x: torch.Tensor) -> bool:
    """Whether no two values of x [T, heads, head_dim] share memory: each stride steps over everything below it.  (A layout
    that interleaves its dimensions otherwise is counted as shared.)"""
    span = 1
    for stride, size in sorted((s, n) for s, n in zip(x.stride(), x.shape) if n > 1):
        if stride < span:
            return False
        span = stride * (size - 1) + span
    return True


def _disjoint(q: torch.Tensor, k: torch.Tensor) -> bool:
    """Whether q and k, [T, heads, head_dim] without shared values of their own, share no memory: one lies behind the other,
    or in the gaps that the other's tokens or heads leave at the same stride (views of a fused projection)."""
    apart = k.data_ptr() - q.data_ptr()
    if apart < 0:
        q, k, apart = k, q, -apart
    apart, rest = divmod(apart, q.element_size())  # k starts so many values behind q
    stride = [max(x.stride(i) if x.shape[i] > 1 else 0 for x in (q, k)) for i in range(3)]
    dims = sorted((i for i in range(3) if stride[i]), key=lambda i: stride[i])

    def reach(x: torch.Tensor) -> int:
        return sum(x.stride(i) * (x.shape[i] - 1) for i in dims if x.shape[i] > 1) + 1

    if apart >= reach(q):
        return True
    while dims and not rest:
        step = dims.pop()  # the widest step: both lie within a stride of it, or are counted as shared
        s = stride[step]
        apart %= s
        if any(x.shape[step] > 1 and x.stride(step) != s for x in (q, k)) or reach(q) > s or apart + reach(k) > s:
            return False
        if apart >= reach(q):
            return True
    return False


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
    Returns new contiguous tensors, or with inplace the given ones, overwritten (q and k must not share memory then, nor
    may tokens or heads of one of them).
    A token at a negative position (padding) is copied unchanged; one behind the table comes out as NaN."""
    lib = _load_ext()
    _require_cuda(q, "q")
    if q.dtype not in _DTYPE_CODE:
        raise RuntimeError("apply_rotary takes float16, bfloat16 or float32")
    if q.dim() != 3 or (k is not None and k.dim() != 3):
        raise ValueError("q and k must be [T, heads, head_dim]")
    dev, dtype = q.device, q.dtype
    t, hq, hd = q.shape
    qs = q.stride()
    hk, ks, kos, k_ptr, ko_ptr = 0, (0, 0, 1), (0, 0), None, None
    if k is not None:
        tk, hk, hdk = k.shape
        ks, k_ptr = k.stride(), k.data_ptr()
        if tk != t or hdk != hd or k.dtype != dtype or k.device != dev:
            raise ValueError("k must match q in tokens, head_dim, dtype and device")
    if hd > 1 and (qs[2] != 1 or ks[2] != 1):
        raise ValueError("q and k must have unit stride in the head")
    if cos_sin.dim() != 3 or cos_sin.shape[2] != 2 or cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous():
        raise ValueError("cos_sin must be a contiguous float32 [positions, rotary_dim / 2, 2] table")
    rd = 2 * cos_sin.shape[1]
    if cos_sin.shape[0] < 1 or not 2 <= rd <= hd or hd > 512:
        raise ValueError("the table must rotate between 2 and head_dim (at most 512) values")
    if positions.dtype not in (torch.int32, torch.int64) or positions.dim() != 1 or positions.shape[0] != t:
        raise ValueError("positions must be int32 or int64 with one value for each token")
    if cos_sin.device != dev or positions.device != dev:
        raise ValueError("q, cos_sin and positions must be on one device")
    if not 1 <= hq <= MAX_HEADS or (k is not None and not 1 <= hk <= MAX_HEADS):
        raise ValueError(f"q and k must have 1 to {MAX_HEADS} heads")
    if inplace and t > 0 and not (_distinct(q) and (k is None or (_distinct(k) and _disjoint(q, k)))):
        raise ValueError("inplace needs q and k whose tokens and heads share no memory, with one another either")
    q_out, k_out = (q, k) if inplace else (_empty((t, hq, hd), dtype, dev), None)
    if k is not None:
        if not inplace:
            k_out = _empty((t, hk, hd), dtype, dev)
        kos, ko_ptr = k_out.stride(), k_out.data_ptr()
    if t > 0:
        pos = positions if positions.is_contiguous() else positions.contiguous()
        qos = q_out.stride()
        rc = _run(
            dev, lib.b200w4a4_rotary, q.data_ptr(), qs[0], qs[1], q_out.data_ptr(), qos[0], qos[1], hq, k_ptr, ks[0], ks[1],
            ko_ptr, kos[0], kos[1], hk, _DTYPE_CODE[dtype], cos_sin.data_ptr(), cos_sin.shape[0], pos.data_ptr(),
            1 if pos.dtype == torch.int64 else 0, t, hd, rd, 1 if interleaved else 0, 1 if inverse else 0, _stream_ptr(dev))
        _lib.check(rc, "rotary")
    return q_out, k_out
