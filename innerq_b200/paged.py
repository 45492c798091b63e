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

import ctypes as C
import math

import torch

from . import _lib
from .prompt import _index, _rows
from .store import D_SUPPORTED, dtype_code, require_cuda, stream_ptr

__all__ = ["PagedCache", "TILE", "BLOCK_BYTES"]

TILE = 32            # tokens of a packed tile
BLOCK_BYTES = 4608   # one tile of one head: codes and scales of keys and values


class PagedCache:
    """The storage: ``pages`` uint8 [n_pages, Hkv, page_size / 32, 4608] and
    ``dense_k`` / ``dense_v`` [n_slots, Hkv, w_sink + w_recent + 32, 128] in
    fp16 or bf16 (16-byte aligned, contiguous; see ``allocate``)."""

    def __init__(self, pages: torch.Tensor, dense_k: torch.Tensor, dense_v: torch.Tensor, w_sink: int, w_recent: int):
        require_cuda(pages, "pages")
        n_slots, hkv, rows, d = dense_k.shape
        if d != D_SUPPORTED:
            raise NotImplementedError(f"head_dim {d} is not built (128 is)")
        if w_sink < 0 or w_recent < 0 or w_sink % TILE or w_recent % TILE:
            raise ValueError(f"sink {w_sink} and recent window {w_recent} must be multiples of {TILE}")
        if rows != w_sink + w_recent + TILE or dense_v.shape != dense_k.shape or dense_v.dtype != dense_k.dtype:
            raise ValueError(f"slots must hold {w_sink + w_recent + TILE} rows of keys and of values, "
                             f"got {tuple(dense_k.shape)} and {tuple(dense_v.shape)}")
        if pages.dtype != torch.uint8 or pages.dim() != 4 or pages.shape[1] != hkv or pages.shape[3] != BLOCK_BYTES:
            raise ValueError(f"pages must be uint8 [pages, {hkv}, tiles, {BLOCK_BYTES}], got {pages.dtype} {tuple(pages.shape)}")
        if not (pages.is_contiguous() and dense_k.is_contiguous() and dense_v.is_contiguous()):
            raise ValueError("pages and slots must be contiguous")
        if not (pages.device == dense_k.device == dense_v.device):
            raise ValueError("pages and slots must be on one device")
        self.pages, self.dense_k, self.dense_v = pages, dense_k, dense_v
        self.w_sink, self.w_recent = w_sink, w_recent
        self.dtype, self.device = dense_k.dtype, pages.device
        self.n_kv_heads, self.page_size = hkv, pages.shape[2] * TILE
        self._c = _lib.Paged(
            C.sizeof(_lib.Paged), dtype_code(dense_k.dtype), d, hkv, pages.shape[2], pages.shape[0], n_slots, w_sink,
            w_recent, 0, 0, pages.data_ptr(), dense_k.data_ptr(), dense_v.data_ptr(), None, 0, None, None)

    @classmethod
    def allocate(cls, n_pages: int, n_kv_heads: int, n_slots: int, page_size: int = 64, w_sink: int = 32,
                 w_recent: int = 96, dtype: torch.dtype = torch.float16, device=None) -> "PagedCache":
        if page_size < TILE or page_size % TILE or page_size > 64 * TILE:
            raise ValueError(f"page_size {page_size} must be a multiple of {TILE} up to {64 * TILE}")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        rows = w_sink + w_recent + TILE
        dense = [torch.empty((n_slots, n_kv_heads, rows, D_SUPPORTED), dtype=dtype, device=device) for _ in range(2)]
        pages = torch.empty((n_pages, n_kv_heads, page_size // TILE, BLOCK_BYTES), dtype=torch.uint8, device=device)
        return cls(pages, dense[0], dense[1], w_sink, w_recent)

    def packed_tokens(self, length: int) -> int:
        """Tokens of a sequence of this length that are held in 4 bits."""
        return max(0, length - self.w_sink - self.w_recent) // TILE * TILE

    def pages_for(self, length: int) -> int:
        """Pages that a sequence of this length needs."""
        return -(-self.packed_tokens(length) // self.page_size)

    # ---------------------------------------------------------------- steps
    def _args(self, page_table, slots, seq_lens) -> _lib.Paged:
        if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != self.device:
            raise TypeError(f"page_table must be int32 [sequences, pages] on {self.device}")
        B, columns = page_table.shape
        if columns > 1 and page_table.stride(1) != 1:
            page_table = page_table.contiguous()
        slots = _index(slots, "slots", B, self.device)
        seq_lens = _index(seq_lens, "seq_lens", B, self.device)
        c = _lib.Paged.from_buffer_copy(self._c)
        c.B, c.max_pages = B, columns
        c.table, c.table_stride = page_table.data_ptr(), page_table.stride(0)
        c.slots, c.seq_lens = slots.data_ptr(), seq_lens.data_ptr()
        c._keep = (page_table, slots, seq_lens)  # copies live until the launch
        return c

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
        position without a row gives NaN.  Without cos and sin nothing is
        rotated.  Returns the rotated q (None without q), with return_k the
        pair (q, rotated k): the 16-bit keys that attention over the prompt
        reads."""
        k = _rows(k, "key", self.dtype, self.device)
        v = _rows(v, "value", self.dtype, self.device)
        T = k.shape[0]
        if k.shape != (T, self.n_kv_heads, D_SUPPORTED) or v.shape != k.shape:
            raise ValueError(f"key {tuple(k.shape)} and value {tuple(v.shape)} must be [tokens, {self.n_kv_heads}, 128]")
        c = self._args(page_table, slots, seq_lens)
        a = _lib.PagedNew()
        a.struct_size, a.T = C.sizeof(_lib.PagedNew), T
        q_out = k_out = None
        if q is not None:
            q = _rows(q, "query", self.dtype, self.device)
            if q.shape[0] != T or q.shape[2] != D_SUPPORTED:
                raise ValueError(f"query {tuple(q.shape)} must be [{T}, heads, 128]")
            q_out = torch.empty(q.shape, dtype=self.dtype, device=self.device)
            a.Hq, a.q, a.q_out = q.shape[1], q.data_ptr(), q_out.data_ptr()
            a.q_st, a.q_sh, _ = q.stride()
            a.qo_st, a.qo_sh = q.shape[1] * D_SUPPORTED, D_SUPPORTED
        a.k, a.v = k.data_ptr(), v.data_ptr()
        a.k_st, a.k_sh, _ = k.stride()
        a.v_st, a.v_sh, _ = v.stride()
        if return_k:
            k_out = torch.empty(k.shape, dtype=self.dtype, device=self.device)
            a.k_out = k_out.data_ptr()
            a.ko_st, a.ko_sh = self.n_kv_heads * D_SUPPORTED, D_SUPPORTED
        if cu_seqlens is not None:
            cu_seqlens = _index(cu_seqlens, "cu_seqlens", c.B + 1, self.device)
            a.cu_seqlens = cu_seqlens.data_ptr()
        elif T != c.B:
            raise ValueError(f"{T} tokens for {c.B} sequences need cu_seqlens")
        if (cos is None) != (sin is None):
            raise ValueError("cos and sin come together")
        if cos is not None:
            cos, sin = self._table(cos), self._table(sin)
            if cos.shape != sin.shape or cos.stride(0) != sin.stride(0):
                raise ValueError(f"cos {tuple(cos.shape)} and sin {tuple(sin.shape)} differ")
            a.rot_dim, a.max_pos, a.cs_stride = 2 * cos.shape[1], cos.shape[0], cos.stride(0)
            a.cos, a.sin = cos.data_ptr(), sin.data_ptr()
            a.interleaved = int(bool(interleaved))
        _lib.call("innerq_paged_append", C.byref(c), C.byref(a), stream_ptr(self.device))
        return (q_out, k_out) if return_k else q_out

    def _table(self, t: torch.Tensor) -> torch.Tensor:
        if t.dim() != 2 or t.dtype != torch.float32 or t.device != self.device:
            raise TypeError(f"cos and sin must be fp32 [positions, rot / 2] on {self.device}")
        if t.stride(1) != 1 or t.stride(0) % 4 or t.data_ptr() % 16:
            t = t.clone(memory_format=torch.contiguous_format)
        return t

    def attend(self, q: torch.Tensor, page_table: torch.Tensor, slots: torch.Tensor, seq_lens: torch.Tensor,
               scale: float | None = None, out: torch.Tensor | None = None,
               lse: torch.Tensor | None = None) -> torch.Tensor:
        """Decode attention: q [B, Hq, 128], one query token per sequence,
        over its seq_lens[b] cached tokens (this step's included) -> out
        [B, Hq, 128].  A sequence without tokens gets zeros.  lse (optional,
        fp32 [B, Hq]): log2-sum-exp2 of the scaled logits."""
        q = _rows(q, "query", self.dtype, self.device)
        c = self._args(page_table, slots, seq_lens)
        B, Hq, D = q.shape
        if B != c.B or D != D_SUPPORTED:
            raise ValueError(f"query {tuple(q.shape)} must be [{c.B}, heads, 128]")
        if out is None:
            out = torch.empty((B, Hq, D), dtype=self.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype != self.dtype or out.device != self.device or out.stride(2) != 1:
            raise ValueError("out must be like the query, with contiguous rows")
        if lse is not None and (lse.shape != (B, Hq) or lse.dtype != torch.float32 or not lse.is_contiguous()
                                or lse.device != self.device):
            raise ValueError("lse must be a contiguous fp32 [sequences, heads] tensor")
        ws_bytes = _lib.load().innerq_paged_attn_workspace(C.byref(c), Hq)
        if ws_bytes < 0:
            raise _lib.InnerqError("innerq_paged_attn_workspace", -1, _lib.last_error())
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=self.device)  # of this stream
        _lib.call("innerq_paged_attn", C.byref(c), Hq, q.data_ptr(), q.stride(0), q.stride(1),
                  float(scale if scale is not None else 1.0 / math.sqrt(D)), ws.data_ptr(), ws_bytes, out.data_ptr(),
                  out.stride(0), out.stride(1), None if lse is None else lse.data_ptr(), stream_ptr(self.device))
        return out

    def read(self, page_table: torch.Tensor, slots: torch.Tensor, seq_lens: torch.Tensor, starts: torch.Tensor,
             cu_seqlens: torch.Tensor, n_tokens: int) -> tuple[torch.Tensor, torch.Tensor]:
        """What the cache holds, dequantized and rounded to the dtype
        (``cache.py:235-281``): token cu_seqlens[b] + i of the results
        [n_tokens, Hkv, 128] is token starts[b] + i of sequence b.  n_tokens is
        cu_seqlens[-1], known to the caller; positions outside a sequence read
        as NaN.  Feeds prompt_attention with the tokens before a chunk."""
        c = self._args(page_table, slots, seq_lens)
        starts = _index(starts, "starts", c.B, self.device)
        cu_seqlens = _index(cu_seqlens, "cu_seqlens", c.B + 1, self.device)
        shape = (n_tokens, self.n_kv_heads, D_SUPPORTED)
        k, v = (torch.empty(shape, dtype=self.dtype, device=self.device) for _ in range(2))
        _lib.call("innerq_paged_read", C.byref(c), starts.data_ptr(), cu_seqlens.data_ptr(), n_tokens, k.data_ptr(),
                  v.data_ptr(), stream_ptr(self.device))
        return k, v
