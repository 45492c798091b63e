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

import torch

from . import _lib

__all__ = ["prompt_attention"]

_host = _lib.host()


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
    defaults to 128 ** -0.5.  Returns out [Tq, Hq, 128] (given: contiguous
    rows, any token and head stride, apart from the inputs); lse (optional, fp32
    [Tq, Hq]) receives the log2-sum-exp2 of the scaled logits.  Rows past
    cu_seqlens[-1] are not written."""
    out = _host.prompt(q, k, v, cu_seqlens, cu_seqlens_k, scale, causal, out, lse)
    if q.shape[0] and cu_seqlens.shape[0] > 1:
        _lib.launch_count[0] += 1
    return out
