"""Causal attention with a sliding window and always-visible first keys (b200w4a4_window_attention), for prompts,
chunks of a prompt on a cache and single tokens.  Its log-sum-exp is the one `attention_qkv.merge_attention` joins."""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib
from .kernels.vdm_w4a4 import _empty, _load_ext, _require_cuda, _run, _stream_ptr

_CODE = {torch.float16: 0, torch.bfloat16: 1}
# from here on a call takes the kernel for prompts, which needs no workspace (kAttnTcMinQueries; a test holds the two together)
PROMPT_QUERIES = 128


def _readable(x: torch.Tensor) -> Tuple[torch.Tensor, Tuple[int, ...]]:
    """x itself and its pitches when the kernel can read it in place (unit stride in the head, 16-byte steps), else a
    copy's.  The pitch of a dimension of one is 0: it is never used."""
    s0, s1, s2, s3 = x.stride()
    if s3 != 1 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        s0, s1, s2, _ = x.stride()
    if (s0 | s1 | s2) & 7:
        n0, n1, n2, _ = x.shape
        s0, s1, s2 = s0 if n0 > 1 else 0, s1 if n1 > 1 else 0, s2 if n2 > 1 else 0
        if (s0 | s1 | s2) & 7:
            x = x.clone(memory_format=torch.contiguous_format)
            s0, s1, s2, _ = x.stride()
    return x, (s0, s1, s2)


def window_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    window: int,
    sinks: int = 0,
    *,
    kv_lens: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    return_lse: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """q [B, Lq, q_heads, head_dim]; k, v [B, Lk, k_heads, head_dim] (fp16 or bf16, head_dim 64 or 128, q_heads a
    multiple of k_heads: query head h reads key head h // (q_heads // k_heads)) -> out [B, Lq, q_heads, head_dim], and
    with return_lse the fp32 log-sum-exp [B, q_heads, Lq] of the scaled scores.

    kv_lens (int32 [B]; None: Lk) are the valid keys of each sequence, the queries its last Lq positions: query i is
    at p = kv_len - Lq + i and sees keys j <= p with j > p - window or j < sinks.  A window of Lk or more is plain
    causal attention.  A query that sees nothing (p < 0) gives 0, and -inf for the log-sum-exp.  Keys that no
    query sees may hold anything, and a value that is not finite in a key that some queries see reaches those alone (a NaN
    in k all of their output, one in v its own column).  scale: by default head_dim ** -0.5.  Scores, sums and outputs are
    held in fp32; the softmax weights are rounded to q's type before they multiply v, which is most of the error beside the
    output's own rounding.  Strides are free where they are multiples of 16 bytes with unit stride in the head; other
    tensors are copied first."""
    lib = _load_ext()
    _require_cuda(q, "q")
    if q.dtype not in _CODE:
        raise RuntimeError("window_attention takes float16 or bfloat16")
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("q must be [B, Lq, q_heads, head_dim] and k, v [B, Lk, k_heads, head_dim]")
    b, lq, hq, hd = q.shape
    lk, hk = k.shape[1], k.shape[2]
    if k.shape[0] != b or k.shape[3] != hd or hd not in (64, 128):
        raise ValueError("k and v must have q's batch and head_dim (64 or 128)")
    if hk < 1 or hq < 1 or hq % hk or hq // hk > 64:
        raise ValueError("q_heads must be a multiple (at most 64 times) of k_heads")
    if max(b, lq, lk, hq) >= 1 << 31:
        raise ValueError("sizes must be below 2^31")
    dev = q.device
    if k.dtype != q.dtype or v.dtype != q.dtype or k.device != dev or v.device != dev:
        raise ValueError("q, k and v must have one dtype and device")
    if window < 1 or sinks < 0:
        raise ValueError("window must be at least 1 and sinks not negative")
    if scale is None:
        scale = hd ** -0.5
    if not scale > 0:
        raise ValueError("scale must be positive")
    if kv_lens is not None:
        if kv_lens.dtype != torch.int32 or kv_lens.dim() != 1 or kv_lens.shape[0] != b or kv_lens.device != dev:
            raise ValueError("kv_lens must be int32 [B] on q's device")
        kv_lens = kv_lens.contiguous()
    out = _empty((b, lq, hq, hd), q.dtype, dev)
    lse = _empty((b, hq, lq), torch.float32, dev) if return_lse else None
    if out.numel() > 0:
        (q, qs), (k, ks), (v, vs) = _readable(q), _readable(k), _readable(v)
        window, sinks = min(window, max(lk, 1)), min(sinks, lk)
        need = 0  # of workspace: only calls of fewer queries split the keys
        if lq < PROMPT_QUERIES:
            need = _run(dev, lib.b200w4a4_window_attention_workspace_bytes, b, lq, lk, hq, hk, hd, window, sinks)
        ws = _empty((need,), torch.uint8, dev) if need else None
        rc = _run(
            dev, lib.b200w4a4_window_attention, q.data_ptr(), *qs, k.data_ptr(), *ks, v.data_ptr(), *vs,
            kv_lens.data_ptr() if kv_lens is not None else None, out.data_ptr(), lse.data_ptr() if lse is not None else None,
            _CODE[q.dtype], b, lq, lk, hq, hk, hd, window, sinks, scale, ws.data_ptr() if ws is not None else None, need,
            _stream_ptr(dev))
        _lib.check(rc, "window_attention")
    return (out, lse) if return_lse else out
