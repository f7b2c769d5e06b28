"""A key / value cache in pages of 64 positions, in halves, eight or four bits, and what is done with it: new positions rounded
into it, positions read back, attention of one new token per sequence over it.

The caller owns the page table (int32 [sequences, pages a sequence]): position p of sequence i is in page `table[i, p // 64]`.
Sequences may share leading pages (a common prompt); `attend(shared_pages=n)` then reads and multiplies them once for the batch.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import JoshuaB200Error, check
from .rope import Rope, rows_arg, stream_of, tensor_arg, vector_arg

PAGE = 64
TYPES = {"f16": 1, "q4_0": 2, "q8_0": 8}


class _Cache(ctypes.Structure):
    _fields_ = [("type", ctypes.c_uint32), ("n_kv", ctypes.c_uint32), ("head_dim", ctypes.c_uint32), ("n_pages", ctypes.c_uint32),
                ("pages", ctypes.c_void_p)]


class PagedCache:
    def __init__(self, kind: str, n_kv: int, head_dim: int, n_pages: int | None = None, device=None, pages: torch.Tensor | None = None):
        """`n_pages` new pages on `device`, or `pages`: uint8 [n_pages, ...] of that size, used as they are."""
        if kind not in TYPES:
            raise JoshuaB200Error(_lib.E_TYPE, f"a cache of {kind!r}: one of {sorted(TYPES)}")
        lib = _lib.lib()
        self.page_bytes = lib.jq_kv_page_bytes(TYPES[kind], n_kv, head_dim)
        if self.page_bytes == 0:
            raise JoshuaB200Error(_lib.E_INVALID, f"a cache of {n_kv} heads of {head_dim}: head_dim 64, 128 or 256")
        if pages is None:
            pages = torch.empty(n_pages, self.page_bytes, dtype=torch.uint8, device=device)
        tensor_arg(pages, "pages", torch.uint8)
        if not pages.is_contiguous() or pages.shape[0] == 0 or pages.numel() != pages.shape[0] * self.page_bytes:
            raise JoshuaB200Error(_lib.E_INVALID, f"pages must be contiguous, [pages, {self.page_bytes}] bytes, not {list(pages.shape)}")
        self.kind, self.n_kv, self.head_dim, self.pages, self.device = kind, n_kv, head_dim, pages, pages.device
        self._c = _Cache(TYPES[kind], n_kv, head_dim, pages.shape[0], pages.data_ptr())
        self._ref = ctypes.addressof(self._c)
        self.bad_pos = torch.zeros(1, dtype=torch.int32, device=pages.device)  # a row or a sequence had no place
        self._bad = self.bad_pos.data_ptr()
        self._append, self._read, self._attend = lib.jq_kv_append_dev, lib.jq_kv_read_dev, lib.jq_attention_paged_dev
        self._scratch: dict = {}

    def _table(self, table):
        tensor_arg(table, "table", torch.int32, self.device)
        if table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
            raise JoshuaB200Error(_lib.E_INVALID, "a page table is [sequences, pages] with contiguous rows")
        if table.shape[0] > 1 and table.stride(0) != table.shape[1]:
            raise JoshuaB200Error(_lib.E_INVALID, "the rows of a page table follow one another")
        return table.data_ptr(), table.shape[0], table.shape[1]

    def append(self, qkv: torch.Tensor, pos: torch.Tensor, table: torch.Tensor, n_q: int, seq: torch.Tensor | None = None,
               rope: Rope | None = None, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 0.0,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Rows [rows, (n_q + 2 n_kv) * head_dim] at positions `pos` of sequences `seq` (None: row i is sequence i): keys and
        values into the cache, the rotated queries [rows, n_q * head_dim] returned."""
        at, stride, rows = rows_arg(qkv, "qkv", (n_q + 2 * self.n_kv) * self.head_dim, self.device)
        if out is None:
            out = torch.empty(rows, n_q * self.head_dim, dtype=torch.float32, device=self.device)
        elif not out.is_contiguous() or out.shape != (rows, n_q * self.head_dim):
            raise JoshuaB200Error(_lib.E_INVALID, f"out must be contiguous, [{rows}, {n_q * self.head_dim}]")
        tensor_arg(out, "out", torch.float32, self.device)
        if rope is not None and rope.device != self.device:
            raise JoshuaB200Error(_lib.E_INVALID, "the rope table is on another device")
        pages, n_seq, per = self._table(table)
        check(self._append(self._ref, rope.ref if rope else None, at, stride, vector_arg(pos, "pos", rows, torch.int32, self.device),
                           vector_arg(seq, "seq", rows, torch.int32, self.device) if seq is not None else None, pages, n_seq, per,
                           rows, n_q, vector_arg(q_norm, "q_norm", self.head_dim, torch.float32, self.device) if q_norm is not None else None,
                           vector_arg(k_norm, "k_norm", self.head_dim, torch.float32, self.device) if k_norm is not None else None,
                           eps, out.data_ptr(), self._bad, stream_of(qkv)))
        return out

    def read(self, pos: torch.Tensor, table: torch.Tensor, seq: torch.Tensor | None = None, out=None):
        """(keys, values) f32 [n_kv, rows, head_dim] of positions `pos` of sequences `seq` (None: row i is sequence i), into
        `out` (a pair of such tensors, [n_kv, at least rows, head_dim]) if given."""
        rows = pos.shape[0]
        if out is None:
            out = torch.empty(2, self.n_kv, rows, self.head_dim, dtype=torch.float32, device=self.device).unbind(0)
        k, v = out
        for t in out:
            tensor_arg(t, "out", torch.float32, self.device)
            if t.dim() != 3 or t.shape[0] != self.n_kv or t.shape[1] < rows or t.shape[2] != self.head_dim or not t.is_contiguous():
                raise JoshuaB200Error(_lib.E_INVALID, f"out must be contiguous, [{self.n_kv}, at least {rows}, {self.head_dim}]")
        if k.shape != v.shape:
            raise JoshuaB200Error(_lib.E_INVALID, "keys and values go to tensors of one shape")
        pages, n_seq, per = self._table(table)
        check(self._read(self._ref, vector_arg(pos, "pos", rows, torch.int32, self.device),
                         vector_arg(seq, "seq", rows, torch.int32, self.device) if seq is not None else None, pages, n_seq, per, rows,
                         k.data_ptr(), v.data_ptr(), self.head_dim, max(k.shape[1], 1) * self.head_dim, self._bad, stream_of(pos)))
        return k, v

    def scratch(self, batch: int, n_q: int, shared_pages: int = 0) -> torch.Tensor:
        """Zeroed scratch for `attend` of such calls, one stream at a time."""
        n = _lib.lib().jq_attention_paged_scratch_bytes(batch, n_q, self.n_kv, self.head_dim, shared_pages)
        return torch.zeros(n // 4 + 4, dtype=torch.float32, device=self.device)

    def attend(self, q: torch.Tensor, lens: torch.Tensor, table: torch.Tensor, n_q: int, scale: float = 0.0, shared_pages: int = 0,
               out: torch.Tensor | None = None, scratch: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of one query row per sequence, [batch, n_q * head_dim], over its first `lens` positions; the first
        `shared_pages` pages are the same for all.  `scratch`: from `scratch()`; by default one a stream, kept with the cache."""
        at, stride, batch = rows_arg(q, "q", n_q * self.head_dim, self.device)
        if out is None:
            out = torch.empty(batch, n_q * self.head_dim, dtype=torch.float32, device=self.device)
        to, out_stride, n = rows_arg(out, "out", n_q * self.head_dim, self.device)
        pages, n_seq, per = self._table(table)
        if n != batch or n_seq != batch:
            raise JoshuaB200Error(_lib.E_INVALID, f"{batch} query rows, {n} rows of out, {n_seq} of the page table")
        stream = stream_of(q)
        if scratch is None:
            key = (stream, batch, n_q, shared_pages)
            scratch = self._scratch.get(key)
            if scratch is None:
                scratch = self._scratch[key] = self.scratch(batch, n_q, shared_pages)
        check(self._attend(self._ref, at, stride, vector_arg(lens, "lens", batch, torch.int32, self.device), pages, batch, per, n_q,
                           scale, shared_pages, to, out_stride, scratch.data_ptr(), self._bad, stream))
        return out

    def check_flags(self) -> None:
        """Raises if a row or a sequence had no place in the cache (synchronises)."""
        if int(self.bad_pos.item()) != 0:
            self.bad_pos.zero_()
            raise JoshuaB200Error(_lib.E_TOO_LARGE, "a position, sequence or page id lay outside the cache")
