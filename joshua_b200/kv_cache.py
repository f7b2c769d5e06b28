"""A key / value cache in pages of 64 positions, in halves, eight or four bits, and what is done with it: new positions rounded
into it, positions read back, attention of one new token per sequence over it.

The caller owns the page table (int32 [sequences, pages a sequence]): position p of sequence i is in page `table[i, p // 64]`.
Sequences may share leading pages (a common prompt); `attend(shared_pages=n)` then reads and multiplies them once for the batch where
that is the faster way.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import JoshuaB200Error, check
from .rope import Rope, _device, _new, _raw_stream, block_arg, device_index, rows_arg, vector_arg

PAGE = 64
SCRATCH_ZEROED = 1024   # bytes at the beginning of a scratch, zero before its first call
_capturing = torch.cuda.is_current_stream_capturing
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
        self._index = device_index(pages, "pages", torch.uint8)
        if not pages.is_contiguous() or pages.shape[0] == 0 or pages.numel() != pages.shape[0] * self.page_bytes:
            raise JoshuaB200Error(_lib.E_INVALID, f"pages must be contiguous, [pages, {self.page_bytes}] bytes, not {list(pages.shape)}")
        self.kind, self.n_kv, self.head_dim, self.pages, self.device = kind, n_kv, head_dim, pages, pages.device
        self._c = _Cache(TYPES[kind], n_kv, head_dim, pages.shape[0], pages.data_ptr())
        self._ref = ctypes.addressof(self._c)
        self.bad_pos = torch.zeros(1, dtype=torch.int32, device=pages.device)  # a row or a sequence had no place
        self._bad = self.bad_pos.data_ptr()
        self._append, self._read, self._attend = lib.jq_kv_append_dev, lib.jq_kv_read_dev, lib.jq_attention_paged_dev
        self._scratch: dict = {}   # by stream: one, as large as the largest call so far
        self._needs: dict = {}     # bytes by call; by stream and call where the stream's scratch has them

    def _table(self, table):
        if not isinstance(table, torch.Tensor) or table.dtype is not torch.int32 or table.get_device() != self._index \
                or table.dim() != 2 or not table.is_contiguous():
            raise JoshuaB200Error(_lib.E_INVALID, f"a page table is contiguous int32 [sequences, pages] on {self.device}")
        return table.data_ptr(), *table.shape

    def append(self, qkv: torch.Tensor, pos: torch.Tensor, table: torch.Tensor, n_q: int, seq: torch.Tensor | None = None,
               rope: Rope | None = None, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 0.0,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Rows [rows, (n_q + 2 n_kv) * head_dim] at positions `pos` of sequences `seq` (None: row i is sequence i): keys and
        values into the cache, the rotated queries [rows, n_q * head_dim] returned."""
        index, hd, i32, f32 = self._index, self.head_dim, torch.int32, torch.float32
        if index != _device():
            with torch.cuda.device(index):
                return self.append(qkv, pos, table, n_q, seq, rope, q_norm, k_norm, eps, out)
        at, stride, rows = rows_arg(qkv, "qkv", (n_q + 2 * self.n_kv) * hd, index)
        if out is None:
            out = _new(rows, n_q * hd, dtype=f32, device=self.device)
            to = out.data_ptr()
        else:
            to = block_arg(out, "out", (rows, n_q * hd), f32, index)
        if rope is not None and rope._index != index:
            raise JoshuaB200Error(_lib.E_INVALID, "the rope table is on another device")
        pages, n_seq, per = self._table(table)
        rc = self._append(self._ref, rope.ref if rope is not None else None, at, stride, vector_arg(pos, "pos", rows, i32, index),
                          None if seq is None else vector_arg(seq, "seq", rows, i32, index), pages, n_seq, per, rows, n_q,
                          None if q_norm is None else vector_arg(q_norm, "q_norm", hd, f32, index),
                          None if k_norm is None else vector_arg(k_norm, "k_norm", hd, f32, index), eps, to, self._bad,
                          _raw_stream(index))
        if rc:
            check(rc)
        return out

    def read(self, pos: torch.Tensor, table: torch.Tensor, seq: torch.Tensor | None = None, out=None):
        """(keys, values) f32 [n_kv, rows, head_dim] of positions `pos` of sequences `seq` (None: row i is sequence i), into
        `out` (a pair of such tensors, [n_kv, at least rows, head_dim]) if given."""
        index, hd, n_kv = self._index, self.head_dim, self.n_kv
        if index != _device():
            with torch.cuda.device(index):
                return self.read(pos, table, seq, out)
        rows = most = pos.size(0) if isinstance(pos, torch.Tensor) and pos.dim() else 0
        at = vector_arg(pos, "pos", rows, torch.int32, index)
        if out is None:
            out = (_new(n_kv, rows, hd, dtype=torch.float32, device=self.device), _new(n_kv, rows, hd, dtype=torch.float32, device=self.device))
            k_at, v_at = out[0].data_ptr(), out[1].data_ptr()
        else:
            most = out[0].size(1) if isinstance(out[0], torch.Tensor) and out[0].dim() == 3 else -1
            if most < rows:
                raise JoshuaB200Error(_lib.E_INVALID, f"out must be two tensors [{n_kv}, at least {rows}, {hd}]")
            k_at, v_at = (block_arg(t, "out", (n_kv, most, hd), torch.float32, index) for t in out)
        pages, n_seq, per = self._table(table)
        rc = self._read(self._ref, at, None if seq is None else vector_arg(seq, "seq", rows, torch.int32, index), pages, n_seq, per,
                        rows, k_at, v_at, hd, (most or 1) * hd, self._bad, _raw_stream(index))
        if rc:
            check(rc)
        return out

    def scratch(self, batch: int, n_q: int, shared_pages: int = 0) -> torch.Tensor:
        """Zeroed scratch for `attend` of such calls, one stream at a time."""
        return torch.zeros(self.scratch_bytes(batch, n_q, shared_pages) // 4 + 4, dtype=torch.float32, device=self.device)

    def scratch_bytes(self, batch: int, n_q: int, shared_pages: int = 0) -> int:
        key = batch, n_q, shared_pages
        if key not in self._needs:
            self._note(key, _lib.lib().jq_attention_paged_scratch_bytes(batch, n_q, self.n_kv, self.head_dim, shared_pages))
        return self._needs[key]

    def _grow(self, stream: int, batch: int, n_q: int, shared_pages: int) -> None:
        """A scratch of the stream for such calls."""
        need, has = self.scratch_bytes(batch, n_q, shared_pages), self._scratch.get(stream)
        if has is None or 4 * has.numel() < need:
            self._scratch[stream] = self.scratch(batch, n_q, shared_pages)
        self._note((stream, batch, n_q, shared_pages), need)

    def _note(self, key, n: int) -> None:
        if len(self._needs) >= 1024:
            self._needs.clear()
        self._needs[key] = n

    def attend(self, q: torch.Tensor, lens: torch.Tensor, table: torch.Tensor, n_q: int, scale: float = 0.0, shared_pages: int = 0,
               out: torch.Tensor | None = None, scratch: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of one query row per sequence, [batch, n_q * head_dim], over its first `lens` positions; the first
        `shared_pages` pages are the same for all.  `scratch`: from `scratch()`, of this call or a larger one; by default one a
        stream, kept with the cache (while a graph is captured, the graph's own)."""
        index, width = self._index, n_q * self.head_dim
        if index != _device():
            with torch.cuda.device(index):
                return self.attend(q, lens, table, n_q, scale, shared_pages, out, scratch)
        at, stride, batch = rows_arg(q, "q", width, index)
        n = batch
        if out is None:
            out = _new(batch, width, dtype=torch.float32, device=self.device)
            to, out_stride = out.data_ptr(), width
        else:
            to, out_stride, n = rows_arg(out, "out", width, index)
        pages, n_seq, per = self._table(table)
        if n != batch or n_seq != batch:
            raise JoshuaB200Error(_lib.E_INVALID, f"{batch} query rows, {n} rows of out, {n_seq} of the page table")
        stream = _raw_stream(index)
        if scratch is None:
            if _capturing():  # the graph's own, its counters zeroed by it: it may be replayed beside this stream's next call
                scratch = _new(self.scratch_bytes(batch, n_q, shared_pages) // 4 + 4, dtype=torch.float32, device=self.device)
                scratch[:SCRATCH_ZEROED // 4].zero_()
            else:
                if (stream, batch, n_q, shared_pages) not in self._needs:
                    self._grow(stream, batch, n_q, shared_pages)
                scratch = self._scratch[stream]
        else:
            need = self.scratch_bytes(batch, n_q, shared_pages)
            if not isinstance(scratch, torch.Tensor) or scratch.get_device() != index or not scratch.is_contiguous() \
                    or scratch.numel() * scratch.element_size() < max(need, 1) or scratch.data_ptr() % 16:
                raise JoshuaB200Error(_lib.E_INVALID, f"scratch must be {need} contiguous bytes on {self.device}, from a 16-byte boundary on")
        rc = self._attend(self._ref, at, stride, vector_arg(lens, "lens", batch, torch.int32, index), pages, batch, per, n_q, scale,
                          shared_pages, to, out_stride, scratch.data_ptr(), self._bad, stream)
        if rc:
            check(rc)
        return out

    def check_flags(self) -> None:
        """Raises if a row or a sequence had no place in the cache (synchronises)."""
        if int(self.bad_pos.item()) != 0:
            self.bad_pos.zero_()
            raise JoshuaB200Error(_lib.E_TOO_LARGE, "a position, sequence or page id lay outside the cache")
