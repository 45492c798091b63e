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
        dshape, pshape = dense_k.shape, pages.shape
        if len(dshape) != 4 or len(pshape) != 4:
            raise ValueError(f"pages {tuple(pshape)} and slots {tuple(dshape)} must have four dimensions")
        n_slots, hkv, rows, d = dshape
        if d != D_SUPPORTED:
            raise NotImplementedError(f"head_dim {d} is not built (128 is)")
        if w_sink < 0 or w_recent < 0 or w_sink % TILE or w_recent % TILE:
            raise ValueError(f"sink {w_sink} and recent window {w_recent} must be multiples of {TILE}")
        dtype = dense_k.dtype
        if rows != w_sink + w_recent + TILE or dense_v.shape != dshape or dense_v.dtype != dtype:
            raise ValueError(f"slots must hold {w_sink + w_recent + TILE} rows of keys and of values, "
                             f"got {tuple(dshape)} and {tuple(dense_v.shape)}")
        if pages.dtype != torch.uint8 or pshape[1] != hkv or pshape[3] != BLOCK_BYTES:
            raise ValueError(f"pages must be uint8 [pages, {hkv}, tiles, {BLOCK_BYTES}], got {pages.dtype} {tuple(pshape)}")
        if not (pages.is_contiguous() and dense_k.is_contiguous() and dense_v.is_contiguous()):
            raise ValueError("pages and slots must be contiguous")
        device = pages.device
        if not (device == dense_k.device == dense_v.device):
            raise ValueError("pages and slots must be on one device")
        self.pages, self.dense_k, self.dense_v = pages, dense_k, dense_v
        self.w_sink, self.w_recent = w_sink, w_recent
        self.dtype, self.device = dtype, device
        self.n_kv_heads, self.page_size = hkv, pshape[2] * TILE
        self._head = (_lib.PAGED_FORMAT.size, dtype_code(dtype), d, hkv, pshape[2], pshape[0], n_slots, w_sink, w_recent)

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
    def _args(self, page_table, slots, seq_lens):
        """(innerq_paged as bytes, number of sequences, tensors that must live
        until the launch)."""
        device = self.device
        if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != device:
            raise TypeError(f"page_table must be int32 [sequences, pages] on {device}")
        B, columns = page_table.shape
        stride, step = page_table.stride()
        if columns > 1 and step != 1:
            page_table = page_table.contiguous()
            stride = columns
        slots = _index(slots, "slots", B, device)
        seq_lens = _index(seq_lens, "seq_lens", B, device)
        c = _lib.PAGED_FORMAT.pack(*self._head, B, columns, self.pages.data_ptr(), self.dense_k.data_ptr(),
                                   self.dense_v.data_ptr(), page_table.data_ptr(), stride, slots.data_ptr(),
                                   seq_lens.data_ptr())
        return c, B, (page_table, slots, seq_lens)

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
        dtype, device, hkv = self.dtype, self.device, self.n_kv_heads
        k, v = _rows(k, "key", dtype, device), _rows(v, "value", dtype, device)
        shape = k.shape
        T = shape[0]
        if shape[1] != hkv or shape[2] != D_SUPPORTED or v.shape != shape:
            raise ValueError(f"key {tuple(shape)} and value {tuple(v.shape)} must be [tokens, {hkv}, 128]")
        c, B, keep = self._args(page_table, slots, seq_lens)
        k_st, k_sh, _ = k.stride()
        v_st, v_sh, _ = v.stride()
        q_out = k_out = None
        Hq = q_ptr = q_st = q_sh = qo_ptr = ko_ptr = 0
        if q is not None:
            q = _rows(q, "query", dtype, device)
            n, Hq, d = q.shape
            if n != T or d != D_SUPPORTED:
                raise ValueError(f"query {tuple(q.shape)} must be [{T}, heads, 128]")
            q_out = q.new_empty((T, Hq, d))
            q_ptr, qo_ptr = q.data_ptr(), q_out.data_ptr()
            q_st, q_sh, _ = q.stride()
        if return_k:
            k_out = k.new_empty(shape)
            ko_ptr = k_out.data_ptr()
        cu = 0
        if cu_seqlens is not None:
            cu_seqlens = _index(cu_seqlens, "cu_seqlens", B + 1, device)
            cu = cu_seqlens.data_ptr()
        elif T != B:
            raise ValueError(f"{T} tokens for {B} sequences need cu_seqlens")
        rot = max_pos = c_ptr = s_ptr = c_stride = 0
        if cos is not None and sin is not None:
            cos, sin = self._table(cos), self._table(sin)
            max_pos, half = cos.shape
            c_stride = cos.stride(0)
            if sin.shape != cos.shape or sin.stride(0) != c_stride:
                cos, sin = cos.contiguous(), sin.contiguous()
                c_stride = half
                if sin.shape != cos.shape:
                    raise ValueError(f"cos {tuple(cos.shape)} and sin {tuple(sin.shape)} differ")
            rot, c_ptr, s_ptr = 2 * half, cos.data_ptr(), sin.data_ptr()
        elif cos is not None or sin is not None:
            raise ValueError("cos and sin come together")
        a = _lib.PAGED_NEW_FORMAT.pack(
            _lib.PAGED_NEW_FORMAT.size, Hq, T, rot, 1 if interleaved else 0, max_pos, q_ptr, q_st, q_sh, k.data_ptr(), k_st,
            k_sh, v.data_ptr(), v_st, v_sh, cu, c_ptr, s_ptr, c_stride, qo_ptr, Hq * D_SUPPORTED, D_SUPPORTED, ko_ptr,
            hkv * D_SUPPORTED, D_SUPPORTED)
        _lib.call("innerq_paged_append", c, a, stream_ptr(device))
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
        dtype, device = self.dtype, self.device
        q = _rows(q, "query", dtype, device)
        c, n, keep = self._args(page_table, slots, seq_lens)
        B, Hq, D = q.shape
        if B != n or D != D_SUPPORTED:
            raise ValueError(f"query {tuple(q.shape)} must be [{n}, heads, 128]")
        if out is None:
            out = q.new_empty((B, Hq, D))
        elif out.shape != q.shape or out.dtype != dtype or out.device != device or out.stride(2) != 1:
            raise ValueError("out must be like the query, with contiguous rows")
        if lse is not None and (lse.shape != (B, Hq) or lse.dtype != torch.float32 or not lse.is_contiguous()
                                or lse.device != device):
            raise ValueError("lse must be a contiguous fp32 [sequences, heads] tensor")
        ws_bytes = _lib.load().innerq_paged_attn_workspace(c, Hq)
        if ws_bytes < 0:
            raise _lib.InnerqError("innerq_paged_attn_workspace", -1, _lib.last_error())
        ws = self.pages.new_empty(ws_bytes)  # bytes of this stream's own
        q_sb, q_sh, _ = q.stride()
        o_sb, o_sh, _ = out.stride()
        _lib.call("innerq_paged_attn", c, Hq, q.data_ptr(), q_sb, q_sh,
                  1.0 / math.sqrt(D) if scale is None else float(scale), ws.data_ptr(), ws_bytes, out.data_ptr(),
                  o_sb, o_sh, None if lse is None else lse.data_ptr(), stream_ptr(device))
        return out

    def read(self, page_table: torch.Tensor, slots: torch.Tensor, seq_lens: torch.Tensor, starts: torch.Tensor,
             cu_seqlens: torch.Tensor, n_tokens: int) -> tuple[torch.Tensor, torch.Tensor]:
        """What the cache holds, dequantized and rounded to the dtype
        (``cache.py:235-281``): token cu_seqlens[b] + i of the results
        [n_tokens, Hkv, 128] is token starts[b] + i of sequence b.  n_tokens is
        cu_seqlens[-1], known to the caller; positions outside a sequence read
        as NaN.  Feeds prompt_attention with the tokens before a chunk."""
        c, B, keep = self._args(page_table, slots, seq_lens)
        starts = _index(starts, "starts", B, self.device)
        cu_seqlens = _index(cu_seqlens, "cu_seqlens", B + 1, self.device)
        shape = (n_tokens, self.n_kv_heads, D_SUPPORTED)
        k, v = self.dense_k.new_empty(shape), self.dense_k.new_empty(shape)
        _lib.call("innerq_paged_read", c, starts.data_ptr(), cu_seqlens.data_ptr(), n_tokens, k.data_ptr(),
                  v.data_ptr(), stream_ptr(self.device))
        return k, v
