"""Attention of whole prompts, packed one behind the other.

``prompt_attention`` is the prefill half of a continuous-batching step: the
prompts (or chunks of prompts) of a scheduling step lie one behind the other
in ``[tokens, heads, 128]`` tensors and each attends to its own keys, causally
and with grouped heads.  The keys of a sequence may be longer than its
queries: the last query lines up with the last key, so a chunk sees the tokens
before it (``PagedCache.read`` gives those of a paged cache).  The reference
prefills through Hugging Face sdpa, one length for the whole batch
(``src/innerq/cache.py:390-392``).
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .store import dtype_code, require_cuda, stream_ptr

__all__ = ["prompt_attention"]


def _rows(t: torch.Tensor, what: str, dtype, device) -> torch.Tensor:
    """t as [tokens, heads, 128] with contiguous, 16-byte aligned rows."""
    if t.dim() != 3:
        raise ValueError(f"{what} must be [tokens, heads, head_dim], got {tuple(t.shape)}")
    if t.dtype != dtype or t.device != device:
        raise TypeError(f"{what} is {t.dtype} on {t.device}, expected {dtype} on {device}")
    st, sh, sd = t.stride()
    if sd != 1 or st % 8 or sh % 8 or t.data_ptr() % 16 or (st == 0 and t.shape[0] > 1) or (sh == 0 and t.shape[1] > 1):
        t = t.contiguous()
        if t.data_ptr() % 16:  # a contiguous view at an odd offset
            t = t.clone()
    return t


def _index(t: torch.Tensor, what: str, n: int | None, device) -> torch.Tensor:
    """An int32 vector on the device (n elements)."""
    if t.dim() != 1 or (n is not None and t.shape[0] != n):
        raise ValueError(f"{what} must have {n} elements, got shape {tuple(t.shape)}")
    if t.dtype != torch.int32 or t.device != device:
        raise TypeError(f"{what} must be int32 on {device}, got {t.dtype} on {t.device}")
    return t if t.stride(0) == 1 else t.contiguous()


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     cu_seqlens_k: torch.Tensor | None = None, scale: float | None = None,
                     causal: bool = True, out: torch.Tensor | None = None,
                     lse: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q k^T * scale) v of packed sequences.

    q [Tq, Hq, 128], k and v [Tk, Hkv, 128] (fp16 or bf16, Hq a multiple of
    Hkv; any token and head stride).  cu_seqlens, cu_seqlens_k: int32
    [B + 1] on the device, ascending from 0: sequence b has the queries
    cu_seqlens[b] .. cu_seqlens[b + 1] and the keys cu_seqlens_k[b] ..
    cu_seqlens_k[b + 1] (default: the same).  causal: query i of nq sees the
    keys j <= i + nk - nq.  A query that sees no key gets zeros.  scale
    defaults to 128 ** -0.5.  Returns out [Tq, Hq, 128]; lse (optional, fp32
    [Tq, Hq]) receives the log2-sum-exp2 of the scaled logits.  Rows past
    cu_seqlens[-1] are not written."""
    require_cuda(q, "query")
    q = _rows(q, "query", q.dtype, q.device)
    dt = dtype_code(q.dtype)
    k, v = _rows(k, "key", q.dtype, q.device), _rows(v, "value", q.dtype, q.device)
    Tq, Hq, D = q.shape
    Tk, Hkv, _ = k.shape
    if k.shape != v.shape or k.shape[2] != D:
        raise ValueError(f"shapes of query {tuple(q.shape)}, key {tuple(k.shape)} and value {tuple(v.shape)}")
    cu = _index(cu_seqlens, "cu_seqlens", None, q.device)
    B = cu.shape[0] - 1
    if B < 0:
        raise ValueError("cu_seqlens must have at least one element")
    cu_k = cu if cu_seqlens_k is None else _index(cu_seqlens_k, "cu_seqlens_k", B + 1, q.device)
    if out is None:
        out = q.new_empty((Tq, Hq, D))
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(2) != 1:
        raise ValueError("out must be like the query, with contiguous rows")
    if lse is not None and (lse.shape != (Tq, Hq) or lse.dtype != torch.float32 or not lse.is_contiguous()
                            or lse.device != q.device):
        raise ValueError("lse must be a contiguous fp32 [tokens, heads] tensor")
    a = _lib.PROMPT_FORMAT.pack(
        _lib.PROMPT_FORMAT.size, dt, D, B, Hq, Hkv, Tq, Tk, 1 if causal else 0,
        1.0 / math.sqrt(D) if scale is None else float(scale), q.data_ptr(), *q.stride()[:2], k.data_ptr(), *k.stride()[:2],
        v.data_ptr(), *v.stride()[:2], cu.data_ptr(), cu_k.data_ptr(), out.data_ptr(), *out.stride()[:2],
        0 if lse is None else lse.data_ptr())
    _lib.call("innerq_prompt_attn", a, stream_ptr(q.device))
    return out
