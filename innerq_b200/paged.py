"""A paged 4-bit cache for continuous batching.

``PagedCache`` holds the keys and values of many sequences of different
lengths.  As in an InnerQ layer with 4-bit symmetric codes, keys are grouped
over channels and values over tokens (``src/innerq/cache.py:87-88``), the
first ``w_sink`` tokens and a recent window stay in 16 bits; here the window
holds ``w_recent`` to ``w_recent + 31`` tokens, the packed tokens lie in pages
that a table names per sequence, and the lengths are device tensors, so one
launch serves a whole batch and can be replayed from a CUDA graph.

The cache keeps no lengths: the caller (a scheduler) owns ``page_table``
[B, columns], ``slots`` [B] and ``seq_lens`` [B], all int32 on the device, and
passes the rows of the sequences of a step.  A sequence of L tokens needs
``pages_for(L)`` pages and one slot.

    cache = PagedCache.allocate(n_pages, n_kv_heads, n_slots)
    # prompts, packed one behind the other (seq_lens: lengths before the call)
    q, k = cache.append(q, k, v, table, slots, zeros, cu_seqlens, cos=cos, sin=sin, return_k=True)
    out = prompt_attention(q, k, v, cu_seqlens)
    # a decode step, one token per sequence
    q = cache.append(q, k, v, table, slots, seq_lens, cos=cos, sin=sin)
    seq_lens += 1
    out = cache.attend(q, table, slots, seq_lens)
"""
from __future__ import annotations

import torch

from . import _lib

__all__ = ["PagedCache", "TILE", "BLOCK_BYTES"]

TILE = 32            # tokens of a packed tile
BLOCK_BYTES = 4608   # one tile of one head: codes and scales of keys and values

_host = _lib.host()


class PagedCache:
    """The storage: ``pages`` uint8 [n_pages, Hkv, page_size / 32, 4608] and
    ``dense_k`` / ``dense_v`` [n_slots, Hkv, w_sink + w_recent + 32, 128] in
    fp16 or bf16 (16-byte aligned, contiguous; see ``allocate``)."""

    def __init__(self, pages: torch.Tensor, dense_k: torch.Tensor, dense_v: torch.Tensor, w_sink: int, w_recent: int):
        _host.check_cache(pages, dense_k, dense_v, w_sink, w_recent)
        self.pages, self.dense_k, self.dense_v = pages, dense_k, dense_v
        self.w_sink, self.w_recent = w_sink, w_recent
        self._c = (pages, dense_k, dense_v, w_sink, w_recent)

    @property
    def dtype(self) -> torch.dtype:
        return self.dense_k.dtype

    @property
    def device(self) -> torch.device:
        return self.pages.device

    @property
    def n_kv_heads(self) -> int:
        return self.dense_k.shape[1]

    @property
    def page_size(self) -> int:
        """Tokens of a page."""
        return self.pages.shape[2] * TILE

    @classmethod
    def allocate(cls, n_pages: int, n_kv_heads: int, n_slots: int, page_size: int = 64, w_sink: int = 32,
                 w_recent: int = 96, dtype: torch.dtype = torch.float16, device=None) -> "PagedCache":
        if page_size < TILE or page_size % TILE or page_size > 64 * TILE:
            raise ValueError(f"page_size {page_size} must be a multiple of {TILE} up to {64 * TILE}")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        rows = w_sink + w_recent + TILE
        dense = [torch.empty((n_slots, n_kv_heads, rows, 128), dtype=dtype, device=device) for _ in range(2)]
        pages = torch.empty((n_pages, n_kv_heads, page_size // TILE, BLOCK_BYTES), dtype=torch.uint8, device=device)
        return cls(pages, dense[0], dense[1], w_sink, w_recent)

    def packed_tokens(self, length: int) -> int:
        """Tokens of a sequence of this length that are held in 4 bits."""
        return max(0, length - self.w_sink - self.w_recent) // TILE * TILE

    def pages_for(self, length: int) -> int:
        """Pages that a sequence of this length needs."""
        return -(-self.packed_tokens(length) // self.page_size)

    # ---------------------------------------------------------------- steps
    def append(self, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
               slots: torch.Tensor, seq_lens: torch.Tensor, cu_seqlens: torch.Tensor | None = None,
               cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, interleaved: bool = False,
               return_k: bool = False):
        """Append new tokens and rotate their queries and keys.

        q [T, Hq, 128] (or None), k and v [T, Hkv, 128], any token and head
        stride.  seq_lens: lengths BEFORE the call.  cu_seqlens (int32
        [B + 1]): the sequences' tokens lie one behind the other; None: one
        token per sequence, T == B.  cos, sin: fp32 [positions, rot / 2]; the
        token at position t is rotated by row t over its first rot channels,
        in pairs (i, i + rot / 2), or (2i, 2i + 1) with interleaved=True; a
        position without a row gives NaN, and so does a token of no sequence
        (of a negative length, or past cu_seqlens[-1]), which changes nothing.
        Without cos and sin nothing is rotated.  Returns the rotated q (None without q), with return_k the
        pair (q, rotated k): the 16-bit keys that attention over the prompt
        reads."""
        out = _host.append(self._c, q, k, v, page_table, slots, seq_lens, cu_seqlens, cos, sin, interleaved, return_k)
        if k.shape[0]:
            _lib.launch_count[0] += 1 if cu_seqlens is None or not seq_lens.shape[0] else 2
        return out

    def attend(self, q: torch.Tensor, page_table: torch.Tensor, slots: torch.Tensor, seq_lens: torch.Tensor,
               scale: float | None = None, out: torch.Tensor | None = None,
               lse: torch.Tensor | None = None) -> torch.Tensor:
        """Decode attention: q [B, Hq, 128], one query token per sequence,
        over its seq_lens[b] cached tokens (this step's included) -> out
        [B, Hq, 128] (given: contiguous rows, any strides, apart from q).  A
        sequence without tokens gets zeros.  lse (optional,
        fp32 [B, Hq]): log2-sum-exp2 of the scaled logits."""
        out = _host.attend(self._c, q, page_table, slots, seq_lens, scale, out, lse)
        if q.shape[0]:
            _lib.launch_count[0] += 2
        return out

    def read(self, page_table: torch.Tensor, slots: torch.Tensor, seq_lens: torch.Tensor, starts: torch.Tensor,
             cu_seqlens: torch.Tensor, n_tokens: int) -> tuple[torch.Tensor, torch.Tensor]:
        """What the cache holds, dequantized and rounded to the dtype
        (``cache.py:235-281``): token cu_seqlens[b] + i of the results
        [n_tokens, Hkv, 128] is token starts[b] + i of sequence b.  n_tokens is
        cu_seqlens[-1], known to the caller; positions outside a sequence read
        as NaN.  Feeds prompt_attention with the tokens before a chunk."""
        out = _host.read(self._c, page_table, slots, seq_lens, starts, cu_seqlens, n_tokens)
        if n_tokens and seq_lens.shape[0]:
            _lib.launch_count[0] += 1
        return out
